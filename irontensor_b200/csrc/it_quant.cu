// C ABI of serving from quantised weights and a quantised key/value cache (declared in include/irontensor_b200.h): argument
// checks, choice of kernels, launches.
#include "capi_common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "fa_decode_q4.cuh"
#include "gemm_i8_sm100.cuh"
#include "kv_q4.cuh"
#include "rope_positions.cuh"

namespace {

it_status check_call(it_ctx* ctx, it_stream* stream, it_dtype dtype) {
  if (ctx == nullptr || stream == nullptr) return fail(IT_ERR_INVALID_ARG, "null context or stream");
  if (dtype != IT_F32 && dtype != IT_BF16) return fail(IT_ERR_PRECISION, "dtype %d is not F32 or BF16", (int)dtype);
  return IT_OK;
}

// What the three cache calls have in common.  *empty: there is nothing to do.
it_status check_cache(it_ctx* ctx, it_stream* stream, it_dtype dtype, int32_t B, int32_t n, int32_t Hkv, int32_t D, int32_t max_len,
                      const void* kc, const void* ks, const void* vc, const void* vs) {
  it_status st = check_call(ctx, stream, dtype);
  if (st != IT_OK) return st;
  if (B < 0 || n < 0 || Hkv < 1 || max_len < 1) return fail(IT_ERR_INVALID_ARG, "bad dimension: batch %d, %d, kv_heads %d, max_len %d", B, n, Hkv, max_len);
  if (D < 8 || D > 128 || (D & 7)) return fail(IT_ERR_UNSUPPORTED_SHAPE, "a quantised cache needs head_dim a multiple of 8 in 8..128, got %d", D);
  if (max_len > 0x7fffffff - 65536) return fail(IT_ERR_UNSUPPORTED_SHAPE, "max_len must be at most 2^31 - 65537");   // positions are stepped over
  if (B == 0) return IT_OK;
  if (kc == nullptr || ks == nullptr || vc == nullptr || vs == nullptr) return fail(IT_ERR_INVALID_ARG, "null cache");
  if (!aligned16(kc) || !aligned16(vc)) return fail(IT_ERR_ALIGNMENT, "codes must be 16-byte aligned");
  const int groups = (D + 31) / 32, unit = 2 * (groups & -groups);   // a position's scales are read together where they are 2 or 4
  if ((reinterpret_cast<uintptr_t>(ks) | reinterpret_cast<uintptr_t>(vs)) & (unit - 1))
    return fail(IT_ERR_ALIGNMENT, "scales must be %d-byte aligned", unit);
  return IT_OK;
}

// The largest frequency of the dimension pairs: 1, or with a base below 1 that of the last pair of all or of the longest section.
double largest_frequency(int D, float base, int n_axes, const int32_t* sections, int per_axis) {
  if (base >= 1.f) return 1.0;
  if (!per_axis) return std::pow(static_cast<double>(base), -(D - 2.0) / D);
  const int n = *std::max_element(sections, sections + n_axes);
  return std::pow(static_cast<double>(base), -(n - 1.0) / n);
}

// Frequencies and axes of the dimension pairs.  64 powers in 64 bits take as long as the launch: the last ones are kept, by value.
const it::RopeAxes& rope_axes(int D, float base, int n_axes, const int32_t* sections, int per_axis) {
  struct Last {
    int D = 0, n_axes = 0, per_axis = 0;
    int32_t sections[4] = {};
    float base = 0.f;
    it::RopeAxes axes;
  };
  thread_local Last last;
  const bool same = last.D == D && last.n_axes == n_axes && last.per_axis == (per_axis != 0) && last.base == base &&
                    std::equal(sections, sections + n_axes, last.sections);
  if (same) return last.axes;
  last.D = D;
  last.n_axes = n_axes;
  last.per_axis = per_axis != 0;
  last.base = base;
  std::copy(sections, sections + n_axes, last.sections);
  int pair = 0;
  for (int a = 0; a < n_axes; ++a)
    for (int j = 0; j < sections[a]; ++j, ++pair) {
      last.axes.freq[pair] = std::pow(static_cast<double>(base), per_axis ? -static_cast<double>(j) / sections[a] : -2.0 * pair / D);
      last.axes.axis[pair] = static_cast<uint8_t>(a);
    }
  for (; pair < 64; ++pair) last.axes.freq[pair] = last.axes.axis[pair] = 0;
  return last.axes;
}

// The grid of the kernels that write and read a cache, and the tokens that a CTA takes at a time (kv_q4.cuh).
it_status cache_grid(int B, int tokens, int Hkv, int D, dim3* grid, int* at_once) {
  const int rows = 256 / (4 * ((D + 31) / 32));
  *at_once = std::clamp(tokens, 1, rows);
  const int per_cta = *at_once * it::KV_ROWS_A_THREAD, heads = rows / *at_once;
  const int64_t pairs = static_cast<int64_t>(B) * Hkv;
  if (pairs > 0x7fffffffLL - 65535 * 64) return fail(IT_ERR_UNSUPPORTED_SHAPE, "batch * kv_heads must be below 2^31");
  if (tokens > 0x7fffffff - per_cta) return fail(IT_ERR_UNSUPPORTED_SHAPE, "too many tokens");
  *grid = dim3(static_cast<unsigned>(std::max(1, (tokens + per_cta - 1) / per_cta)), static_cast<unsigned>(std::min<int64_t>((pairs + heads - 1) / heads, 65535)), 2);
  return IT_OK;
}

// f(groups of 32 columns as a constant)
template <typename F>
it_status by_groups(int D, F&& f) {
  switch ((D + 31) / 32) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    default: return f(std::integral_constant<int, 4>{});
  }
}

// How many clusters of `size` CTAs of a kernel are resident at once (asked once per kernel, device and size).
template <typename Kernel>
int clusters_at_once(Kernel kernel, int size, int threads, int smem_bytes, std::atomic<int>& known) {
  if (known == 0) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem_bytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(size);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
    known = n;
  }
  return known;
}

// How 4-bit attention shares out its work (see fa_decode_q4.cuh): clusters of 1, 2, 4 or 8 CTAs a pair, or even shares.  The lengths are
// on the device, so this goes by max_len.  In us, for bf16 at head_dim 128, a fit: a launch of clusters is 4.5, 0.3 for each doubling
// of the cluster and a round of 256 keys 1.25 for a CTA that has an SM for itself, 2.2 for two on one (in clusters of 1, 2, 4 and 8:
// B8 H32/8, 4000 positions, 23.7, 15.7, 16.1 and 22.9; B1 H32/8, 16000: 77, 42.7, 24.5 and 15.4; B4 H16/4, 1000: 8.2, 7.0, 5.8 and 6.9).
// An even launch is 13.5 and its rounds.  The 13.5 is the fit's intercept, over caches that are as full as they may be: launch, scan,
// merge, and the least share, 16 units, which leaves most CTAs of a short launch without work (B1 H32/8, 4000 positions: 13.4, in
// clusters 7.4); 100 positions in a cache of 131072 take 6.9.  (One sequence of 131000, H16/2: 22.4, in clusters of 8 90; B32 H32/8
// ragged to 8190: 47.7, in clusters 69, 56, 55 and 77; 64 pairs of 4000: 20.4 and 15.7.)  Batches are counted as three quarters full
// there, because in clusters the longest sequence decides.  What going by max_len costs: B4 H16/4 ragged to 1000 takes 5.6 in a cache of
// 1024 positions and 12.9 in one of 131072, where clusters of 8 would take 6.6.
template <typename AtOnce>
void choose_decode_q4_plan(long long pairs, int B, int max_len, int sm_count, int per_sm, int groups, AtOnce&& at_once, int* n_splits, bool* even) {
  const double width = 0.35 + 0.65 * groups / 4, two = 2.2 * width, one = per_sm == 1 ? two : 1.25 * width;
  double best = 1e30;
  for (int n = 1; n <= 8; n *= 2) {
    const long long rounds = (static_cast<long long>(max_len) + 256LL * n - 1) / (256LL * n), resident = std::max(1, at_once(n));
    const double round = pairs * n > sm_count ? two : one;
    const double t = 4.5 + 0.3 * (n >= 8 ? 3 : n / 2) + static_cast<double>((pairs + resident - 1) / resident) * rounds * round;
    if (t < best) {
      best = t;
      *n_splits = n;
    }
  }
  const double rounds = static_cast<double>(pairs) * (max_len + 32.0 * it::DQ_START) / (256.0 * per_sm * sm_count);
  const bool countable = static_cast<double>(pairs) * (max_len / 32 + it::DQ_START + 1) < 2e9;   // the shares are counted in 32 bits
  *even = countable && 13.5 + (B > 1 ? 0.75 : 1.0) * rounds * two < best;
}

// Floats of the parts that a persistent attention launch leaves: outputs, then maxima and sums.
size_t decode_q4_part_floats(int D) { return static_cast<size_t>(2 * it::DQ_MAX_CTAS * 8) * (32 * ((D + 31) / 32) + 2); }

it::KvQ4 half_of(const void* codes, const void* scales) {
  return it::KvQ4{static_cast<uint32_t*>(const_cast<void*>(codes)), static_cast<__nv_bfloat16*>(const_cast<void*>(scales))};
}

}  // namespace

extern "C" {

it_status it_rope_positions(it_ctx* ctx, it_stream* stream, it_dtype dtype, int32_t B, int32_t S, int32_t H, int32_t Hkv, int32_t D,
                            float rope_base, int32_t n_axes, const int32_t* sections, int32_t per_axis, int32_t inverse,
                            const int32_t* positions, const void* q_in, const void* k_in, void* q_out, void* k_out) {
  it_status st = check_call(ctx, stream, dtype);
  if (st != IT_OK) return st;
  if (B < 0 || S < 0 || H < 0 || Hkv < 0) return fail(IT_ERR_INVALID_ARG, "negative dimension");
  if (D < 2 || D > 128 || (D & 1)) return fail(IT_ERR_UNSUPPORTED_SHAPE, "rotary embedding needs an even head_dim in 2..128, got %d", D);
  if (!(rope_base > 0.f) || !std::isfinite(rope_base)) return fail(IT_ERR_INVALID_ARG, "rotary base must be positive and finite");
  if (n_axes < 1 || n_axes > 4 || sections == nullptr) return fail(IT_ERR_INVALID_ARG, "1 to 4 axes with a section each, got %d", n_axes);
  int pairs = 0;
  for (int a = 0; a < n_axes; ++a) {
    if (sections[a] < 0 || sections[a] > D / 2 - pairs) return fail(IT_ERR_INVALID_ARG, "sections must add up to head_dim / 2 = %d", D / 2);
    pairs += sections[a];
  }
  if (pairs != D / 2) return fail(IT_ERR_INVALID_ARG, "sections must add up to head_dim / 2 = %d", D / 2);
  if (!(largest_frequency(D, rope_base, n_axes, sections, per_axis) <= it::ROPE_MOST_FREQ))
    return fail(IT_ERR_INVALID_ARG, "rotary base %g makes frequencies above %g", static_cast<double>(rope_base), it::ROPE_MOST_FREQ);
  const int64_t rows = static_cast<int64_t>(B) * S;
  if (rows == 0 || (H == 0 && Hkv == 0)) return IT_OK;
  if (static_cast<int64_t>(H) + Hkv > 65535) return fail(IT_ERR_UNSUPPORTED_SHAPE, "heads + kv_heads must be at most 65535");
  if (positions == nullptr) return fail(IT_ERR_INVALID_ARG, "null positions");
  if (H > 0 && (q_in == nullptr || q_out == nullptr)) return fail(IT_ERR_INVALID_ARG, "null q tensor");
  if (Hkv > 0 && (k_in == nullptr || k_out == nullptr)) return fail(IT_ERR_INVALID_ARG, "null k tensor");
  IT_CUDA(cudaSetDevice(ctx->device));
  const it::RopeAxes& axes = rope_axes(D, rope_base, n_axes, sections, per_axis);
  const int half = D / 2, elem = dtype == IT_F32 ? 4 : 2;
  const bool chunks = (D * elem) % 16 == 0 && aligned16(q_in) && aligned16(q_out) && aligned16(k_in) && aligned16(k_out);
  const uintptr_t pair_mask = 2 * elem - 1;
  if (!chunks && ((reinterpret_cast<uintptr_t>(q_in) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_in) |
                   reinterpret_cast<uintptr_t>(k_out)) & pair_mask))
    return fail(IT_ERR_ALIGNMENT, "q and k must be aligned to a pair of elements");
  // as many tokens a CTA as have two sines per thread and eight chunks, as long as that leaves four CTAs per SM (2 x 4093 tokens of 16 + 4 heads
  // of 128 in bf16, tensors that left L2: 14.8 us, 5.7 TB/s; 8 x 600 of 32 + 8: 16.7, 5.9 TB/s)
  const int token_chunks = (H + Hkv) * (chunks ? D * elem / 16 : half);
  const int n_pos = static_cast<int>(std::clamp<int64_t>(rows / (4LL * ctx->sm_count), 1, std::clamp(2048 / token_chunks, 1, 512 / half)));
  const int64_t ctas = (rows + n_pos - 1) / n_pos;
  if (ctas > 2147483647LL) return fail(IT_ERR_UNSUPPORTED_SHAPE, "too many tokens");
  auto launch = [&](auto kernel, auto* q, auto* k, auto* qo, auto* ko) -> it_status {
    IT_CUDA(launch_dependent(kernel, static_cast<unsigned>(ctas), 256, 0, stream->s, q, k, qo, ko, positions, static_cast<long long>(rows), n_pos,
                             H, Hkv, D, inverse ? 1 : 0, axes));
    ctx->launches += 1;
    return IT_OK;
  };
  if (dtype == IT_F32)
    return launch(chunks ? it::rope_positions_kernel<float, 4> : it::rope_positions_kernel<float, 2>, static_cast<const float*>(q_in),
                  static_cast<const float*>(k_in), static_cast<float*>(q_out), static_cast<float*>(k_out));
  using BF = __nv_bfloat16;
  return launch(chunks ? it::rope_positions_kernel<BF, 8> : it::rope_positions_kernel<BF, 2>, static_cast<const BF*>(q_in),
                static_cast<const BF*>(k_in), static_cast<BF*>(q_out), static_cast<BF*>(k_out));
}

it_status it_kv_cache_q4_append(it_ctx* ctx, it_stream* stream, it_dtype dtype, int32_t B, int32_t T, int32_t Hkv, int32_t D,
                                int32_t max_len, const void* k, const void* v, const int32_t* lengths, const int32_t* counts,
                                int32_t* new_lengths, void* k_codes, void* k_scales, void* v_codes, void* v_scales) {
  it_status st = check_cache(ctx, stream, dtype, B, T, Hkv, D, max_len, k_codes, k_scales, v_codes, v_scales);
  if (st != IT_OK || B == 0) return st;
  if (lengths == nullptr || new_lengths == nullptr) return fail(IT_ERR_INVALID_ARG, "null lengths");
  if (lengths == new_lengths || counts == new_lengths) return fail(IT_ERR_INVALID_ARG, "new_lengths must be another array than lengths and counts");
  if (T > 0 && (k == nullptr || v == nullptr)) return fail(IT_ERR_INVALID_ARG, "null tensor");
  if (!aligned16(k) || !aligned16(v)) return fail(IT_ERR_ALIGNMENT, "k and v must be 16-byte aligned");
  dim3 grid;
  int at_once;
  if ((st = cache_grid(B, T, Hkv, D, &grid, &at_once)) != IT_OK) return st;
  IT_CUDA(cudaSetDevice(ctx->device));
  // Two to three rounds of CTAs, each of which then goes on to other tokens: 8 x 2999 tokens of 8 heads of 128, all of them or padded to half,
  // 23.8 and 14.9 us (in fp32 37.4 and 22.5); with 8 CTAs an SM 26 and 15.3, with one for every 64 tokens 26 and 19.3.
  grid.x = std::min<unsigned>(grid.x, std::max(1u, 12u * static_cast<unsigned>(ctx->sm_count) / (2 * grid.y)));
  auto launch = [&](auto kernel, auto* kk, auto* vv) -> it_status {
    IT_CUDA(launch_dependent(kernel, grid, 256, 0, stream->s, kk, vv, half_of(k_codes, k_scales), half_of(v_codes, v_scales), lengths, counts,
                             new_lengths, B, T, Hkv, D, max_len, at_once, ctx->range_status()));
    ctx->launches += 1;
    return IT_OK;
  };
  return by_groups(D, [&](auto ng) {
    constexpr int NG = decltype(ng)::value;
    const bool full = at_once == 256 / (4 * NG);
    using BF = __nv_bfloat16;
    return dtype == IT_F32 ? launch(full ? it::kv_q4_append_kernel<float, NG, true> : it::kv_q4_append_kernel<float, NG, false>,
                                    static_cast<const float*>(k), static_cast<const float*>(v))
                           : launch(full ? it::kv_q4_append_kernel<BF, NG, true> : it::kv_q4_append_kernel<BF, NG, false>,
                                    static_cast<const BF*>(k), static_cast<const BF*>(v));
  });
}

it_status it_kv_cache_q4_read(it_ctx* ctx, it_stream* stream, it_dtype dtype, int32_t B, int32_t T, int32_t Hkv, int32_t D, int32_t max_len,
                              const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, const int32_t* starts,
                              const int32_t* lengths, void* k, void* v) {
  it_status st = check_cache(ctx, stream, dtype, B, T, Hkv, D, max_len, k_codes, k_scales, v_codes, v_scales);
  if (st != IT_OK || B == 0 || T == 0) return st;
  if (k == nullptr || v == nullptr) return fail(IT_ERR_INVALID_ARG, "null tensor");
  if (!aligned16(k) || !aligned16(v)) return fail(IT_ERR_ALIGNMENT, "k and v must be 16-byte aligned");
  dim3 grid;
  int at_once;
  if ((st = cache_grid(B, T, Hkv, D, &grid, &at_once)) != IT_OK) return st;
  IT_CUDA(cudaSetDevice(ctx->device));
  auto launch = [&](auto kernel, auto* kk, auto* vv) -> it_status {
    IT_CUDA(launch_dependent(kernel, grid, 256, 0, stream->s, kk, vv, half_of(k_codes, k_scales), half_of(v_codes, v_scales), starts, lengths, B, T,
                             Hkv, D, max_len, at_once));
    ctx->launches += 1;
    return IT_OK;
  };
  return by_groups(D, [&](auto ng) {
    constexpr int NG = decltype(ng)::value;
    using BF = __nv_bfloat16;
    return dtype == IT_F32 ? launch(it::kv_q4_read_kernel<float, NG>, static_cast<float*>(k), static_cast<float*>(v))
                           : launch(it::kv_q4_read_kernel<BF, NG>, static_cast<BF*>(k), static_cast<BF*>(v));
  });
}

it_status it_attention_decode_q4_workspace_bytes(int32_t B, int32_t H, int32_t D, size_t* out_bytes) {
  if (out_bytes == nullptr) return fail(IT_ERR_INVALID_ARG, "out_bytes is null");
  if (B < 0 || H < 0) return fail(IT_ERR_INVALID_ARG, "negative dimension");
  if (D < 8 || D > 128 || (D & 7)) return fail(IT_ERR_UNSUPPORTED_SHAPE, "a quantised cache needs head_dim a multiple of 8 in 8..128, got %d", D);
  *out_bytes = (decode_q4_part_floats(D) + B + 2) * 4 / 256 * 256 + 512;
  return IT_OK;
}

it_status it_attention_decode_q4(it_ctx* ctx, it_stream* stream, it_dtype dtype, int32_t B, int32_t H, int32_t Hkv, int32_t D,
                                 int32_t max_len, const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                                 const void* v_scales, const int32_t* lengths, void* o, float* lse, void* workspace,
                                 size_t workspace_bytes) {
  it_status st = check_cache(ctx, stream, dtype, B, H, Hkv, D, max_len, k_codes, k_scales, v_codes, v_scales);
  if (st != IT_OK) return st;
  if (H % Hkv != 0) return fail(IT_ERR_INVALID_ARG, "heads (%d) must be divisible by kv_heads (%d)", H, Hkv);
  if (static_cast<int64_t>(B) * H > 65535) return fail(IT_ERR_UNSUPPORTED_SHAPE, "batch*heads must be <= 65535, got %lld", (long long)B * H);
  if (B == 0 || H == 0) return IT_OK;
  if (q == nullptr || o == nullptr || lengths == nullptr) return fail(IT_ERR_INVALID_ARG, "null tensor");
  if (!aligned16(q) || !aligned16(o)) return fail(IT_ERR_ALIGNMENT, "q and o must be 16-byte aligned");
  size_t need = 0;
  it_attention_decode_q4_workspace_bytes(B, H, D, &need);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(IT_ERR_INVALID_ARG, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return fail(IT_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
  IT_CUDA(cudaSetDevice(ctx->device));
  it::DecodeQ4Params p;
  p.q = q;
  p.k_codes = static_cast<const uint32_t*>(k_codes);
  p.v_codes = static_cast<const uint32_t*>(v_codes);
  p.k_scales = static_cast<const __nv_bfloat16*>(k_scales);
  p.v_scales = static_cast<const __nv_bfloat16*>(v_scales);
  p.lengths = lengths;
  p.o = o;
  p.lse = lse;
  p.status = ctx->range_status();
  p.H = H;
  p.Hkv = Hkv;
  p.D = D;
  p.max_len = max_len;
  p.scale_log2 = (1.0f / sqrtf(static_cast<float>(D))) * 1.4426950408889634f;
  p.B = B;
  const int G = H / Hkv;
  const bool wide = dtype == IT_BF16 && G > 8;
  const int heads = wide ? 16 : 8, chunks = (G + heads - 1) / heads;
  const long long pairs = static_cast<long long>(B) * Hkv * chunks;
  float* ws = static_cast<float*>(workspace);
  p.part_o = ws;
  p.part_ml = ws + static_cast<size_t>(2 * it::DQ_MAX_CTAS * 8) * (32 * ((D + 31) / 32));
  p.units = reinterpret_cast<int*>(ws + decode_q4_part_floats(D));
  int n = 1;
  bool even = false;
  auto main_launch = [&](auto ng, auto terms, auto hd, auto paired) -> it_status {
    constexpr int NG = decltype(ng)::value, TERMS = decltype(terms)::value, HEADS = decltype(hd)::value;
    constexpr bool PAIRED = decltype(paired)::value;
    constexpr int warps = it::dq_warps(TERMS, HEADS, it::PLAN_CLUSTER), even_warps = it::dq_warps(TERMS, HEADS, it::PLAN_EVEN);
    constexpr int bytes = warps * it::DecodeQ4Stage<NG>::WARP_BYTES, even_bytes = even_warps * it::DecodeQ4Stage<NG>::WARP_BYTES;
    static std::atomic<bool> attr_set[16];
    if (!attr_set[ctx->device & 15]) {
      IT_CUDA(cudaFuncSetAttribute(it::fa_decode_q4_kernel<NG, TERMS, HEADS, PAIRED, it::PLAN_CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      IT_CUDA(cudaFuncSetAttribute(it::fa_decode_q4_kernel<NG, TERMS, HEADS, PAIRED, it::PLAN_EVEN>, cudaFuncAttributeMaxDynamicSharedMemorySize, even_bytes));
      attr_set[ctx->device & 15] = true;
    }
    const auto in_clusters = it::fa_decode_q4_kernel<NG, TERMS, HEADS, PAIRED, it::PLAN_CLUSTER>;
    static std::atomic<int> at_once[16][9];
    choose_decode_q4_plan(pairs, B, max_len, ctx->sm_count, it::dq_ctas(TERMS, HEADS, it::PLAN_CLUSTER), NG,
                          [&](int size) { return clusters_at_once(in_clusters, size, 32 * warps, bytes, at_once[ctx->device & 15][size]); }, &n, &even);
    p.n_splits = n;
    const dim3 grid = even ? dim3(std::min(it::dq_ctas(TERMS, HEADS, it::PLAN_EVEN) * ctx->sm_count, wide ? it::DQ_MAX_CTAS / 2 : it::DQ_MAX_CTAS)) : dim3(n, Hkv * chunks, B);
    if (!even) {
      IT_CUDA(launch_cluster(in_clusters, grid, 32 * warps, bytes, stream->s, n, p));
      ctx->launches += 1;
      return IT_OK;
    }
    IT_CUDA(launch_dependent(it::fa_decode_q4_kernel<NG, TERMS, HEADS, PAIRED, it::PLAN_EVEN>, grid, 32 * even_warps, even_bytes, stream->s, p));
    using ST = typename std::conditional<TERMS == 1, __nv_bfloat16, float>::type;
    const bool few = B * H < ctx->sm_count;
    IT_CUDA(launch_dependent(few ? it::fa_decode_q4_merge_kernel<ST, NG, HEADS, 1> : it::fa_decode_q4_merge_kernel<ST, NG, HEADS, NG>,
                             dim3(B * H, few ? NG : 1), 32 * it::DQ_MERGE_WARPS, 0, stream->s, p));
    ctx->launches += 2;
    return IT_OK;
  };
  using one = std::integral_constant<int, 1>;
  using three = std::integral_constant<int, 3>;
  using eight = std::integral_constant<int, 8>;
  return by_groups(D, [&](auto ng) {
    if (dtype == IT_F32) return main_launch(ng, three{}, eight{}, std::false_type{});
    if (wide) return main_launch(ng, one{}, std::integral_constant<int, 16>{}, std::false_type{});
    return G <= 4 ? main_launch(ng, one{}, eight{}, std::true_type{}) : main_launch(ng, one{}, eight{}, std::false_type{});
  });
}

it_status it_quantize_rows_i8(it_ctx* ctx, it_stream* stream, it_dtype dtype, int32_t rows, int32_t cols, const void* x, int8_t* codes,
                              float* scales) {
  it_status st = check_call(ctx, stream, dtype);
  if (st != IT_OK) return st;
  if (rows < 0 || cols < 0) return fail(IT_ERR_INVALID_ARG, "negative dimension");
  if (cols > 0x7fffffff - 65536) return fail(IT_ERR_UNSUPPORTED_SHAPE, "too many columns");
  if (cols == 0 || (cols & 15)) return fail(IT_ERR_UNSUPPORTED_SHAPE, "rows to quantise need a multiple of 16 columns, got %d", cols);
  if (rows == 0) return IT_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr) return fail(IT_ERR_INVALID_ARG, "null tensor");
  if (!aligned16(x) || !aligned16(codes)) return fail(IT_ERR_ALIGNMENT, "x and codes must be 16-byte aligned");
  IT_CUDA(cudaSetDevice(ctx->device));
  // Warps of a row: one where that makes as many warps as keep the memory busy, and as many as a short row has work for
  const int vec = dtype == IT_F32 ? 4 : 8;
  int warps = 1;
  while (warps < 8 && (static_cast<int64_t>(rows) * warps < 16LL * ctx->sm_count || cols > 8 * 32 * vec * warps) && cols > 32 * vec * warps) warps *= 2;
  auto launch = [&](auto kernel, auto* src) -> it_status {
    IT_CUDA(launch_dependent(kernel, static_cast<unsigned>((static_cast<int64_t>(rows) * warps + 7) / 8), 256, 0, stream->s, src, codes, scales, rows,
                             cols));
    ctx->launches += 1;
    return IT_OK;
  };
  auto by_warps = [&](auto* src) -> it_status {
    using ST = std::remove_const_t<std::remove_pointer_t<decltype(src)>>;
    return warps == 1 ? launch(it::quantize_rows_kernel<ST, 1>, src) : warps == 2 ? launch(it::quantize_rows_kernel<ST, 2>, src)
           : warps == 4 ? launch(it::quantize_rows_kernel<ST, 4>, src) : launch(it::quantize_rows_kernel<ST, 8>, src);
  };
  return dtype == IT_F32 ? by_warps(static_cast<const float*>(x)) : by_warps(static_cast<const __nv_bfloat16*>(x));
}

}  // extern "C"

namespace {

// [rows, cols] as TMA sees them: boxes of 128 bytes by `box_rows` rows, 128-byte swizzle, zeros outside.
it_status make_rows_map(it_ctx* ctx, CUtensorMap* map, CUtensorMapDataType type, int bytes, const void* base, int rows, int cols, int box_rows) {
  const cuuint64_t n = static_cast<cuuint64_t>(rows), c = static_cast<cuuint64_t>(cols);
  const cuuint64_t dims[4] = {c, n, 1, 1}, strides[3] = {c * bytes, c * n * bytes, c * n * bytes};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(128 / bytes), static_cast<cuuint32_t>(box_rows), 1, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult r = ctx->encode(map, type, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? IT_OK : fail(IT_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", static_cast<int>(r));
}

template <int BN, int CG, typename OT>
it_status launch_gemm_i8(it_ctx* ctx, cudaStream_t s, const it::GemmI8Params& p) {
  using T = it::GemmI8Traits<BN, CG>;
  it::GemmI8Maps maps;
  it_status st;
  if ((st = make_rows_map(ctx, &maps.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.x, p.M, p.K, T::BM)) != IT_OK) return st;
  if ((st = make_rows_map(ctx, &maps.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.w, p.N, p.K, T::B_ROWS)) != IT_OK) return st;
  const auto type = sizeof(OT) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int r = 2; r >= 0; --r) {
    const int width = p.out.end[r] - (r > 0 ? p.out.end[r - 1] : 0);
    if (width > 0 && (st = make_rows_map(ctx, &maps.out[r], type, sizeof(OT), p.out.ptr[r], p.M, width, 32)) != IT_OK) return st;
    if (width == 0) maps.out[r] = maps.a;   // never used
  }
  static std::atomic<bool> attr_set[16];
  if (!attr_set[ctx->device & 15]) {
    IT_CUDA(cudaFuncSetAttribute(it::gemm_i8_sm100_kernel<BN, CG, OT>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM_BYTES));
    attr_set[ctx->device & 15] = true;
  }
  const long long tiles = static_cast<long long>((p.M + CG * T::BM - 1) / (CG * T::BM)) * ((p.N + BN - 1) / BN);
  const int grid = static_cast<int>(std::min<long long>(tiles, ctx->sm_count / CG)) * CG;
  IT_CUDA(launch_cluster(it::gemm_i8_sm100_kernel<BN, CG, OT>, grid, T::THREADS, T::SMEM_BYTES, s, CG, maps, p));
  ctx->launches += 1;
  return IT_OK;
}

// Up to 16 tokens stream the weights (gemm_i8_skinny_kernel; 16 x 4096 -> 12288: 17.6 us, in 128-column tiles 20.6; 32 x 4096 -> 4096:
// 10.8 and, in 64-column tiles, 8.8).  Above that the tile is the one with the least 4 + waves * (a + b K / 1024) us, fitted to
// 300 x 4096 -> 12288 (27, 21, 23 and 29 us with 64, 128 and 256 columns and pairs of CTAs of 256 x 256), 512 x 4096 -> 4096 (15, 12, 17
// and 17), 2999 x 2048 -> 6144 (52, 35, 31 and 33), 8192 x 4096 -> 12288 (488, 338, 306 and 249: 3.3 POP/s), 8192 x 512 -> 1536 (20, 20,
// 18 and 20).
template <typename OT>
it_status launch_linear_i8(it_ctx* ctx, cudaStream_t s, const it::GemmI8Params& p) {
  if (p.M <= 16) {
    const auto kernel = p.M <= 8 ? it::gemm_i8_skinny_kernel<1, OT> : it::gemm_i8_skinny_kernel<2, OT>;
    IT_CUDA(launch_dependent(kernel, static_cast<unsigned>((p.N + 15) / 16), 256, 0, s, p));
    ctx->launches += 1;
    return IT_OK;
  }
  auto cost = [&](int rows, int columns, int at_once, double a, double b) {
    const long long tiles = static_cast<long long>((p.M + rows - 1) / rows) * ((p.N + columns - 1) / columns);
    return static_cast<double>((tiles + at_once - 1) / at_once) * (a + b * p.K / 1024.0);
  };
  const double c64 = cost(128, 64, ctx->sm_count, 1.0, 1.1), c128 = cost(128, 128, ctx->sm_count, 2.0, 1.45), c256 = cost(128, 256, ctx->sm_count, 3.6, 2.6);
  const double c_pair = cost(256, 256, std::max(1, ctx->sm_count / 2), 4.5, 1.9), best = std::min(std::min(c64, c128), std::min(c256, c_pair));
  if (best == c64) return launch_gemm_i8<64, 1, OT>(ctx, s, p);
  if (best == c128) return launch_gemm_i8<128, 1, OT>(ctx, s, p);
  if (best == c256) return launch_gemm_i8<256, 1, OT>(ctx, s, p);
  return launch_gemm_i8<256, 2, OT>(ctx, s, p);
}

}  // namespace

extern "C" it_status it_linear_i8_fwd(it_ctx* ctx, it_stream* stream, it_dtype out_dtype, int32_t n, int32_t in_dim, int32_t out_dim,
                                      const int8_t* x_codes, const float* x_scales, const int8_t* w_codes, const float* w_scales,
                                      int32_t n_outs, const int32_t* widths, void* const* outs) {
  it_status st = check_call(ctx, stream, out_dtype);
  if (st != IT_OK) return st;
  if (n < 0 || in_dim < 0 || out_dim < 0) return fail(IT_ERR_INVALID_ARG, "negative dimension");
  if (n > 0x7fffffff - 65536 || out_dim > 0x7fffffff - 65536) return fail(IT_ERR_UNSUPPORTED_SHAPE, "n and out_dim must be at most 2^31 - 65537");
  if (in_dim < 16 || in_dim > 65536 || (in_dim & 15))
    return fail(IT_ERR_UNSUPPORTED_SHAPE, "in_dim must be a multiple of 16 in 16..65536, got %d", in_dim);
  if (n_outs < 1 || n_outs > 3 || widths == nullptr || outs == nullptr) return fail(IT_ERR_INVALID_ARG, "1 to 3 results, got %d", n_outs);
  it::GemmI8Params p{};
  int64_t end = 0;
  for (int r = 0; r < 3; ++r) {
    const int width = r < n_outs ? widths[r] : 0;
    if (width < 0) return fail(IT_ERR_INVALID_ARG, "negative width");
    if (width & 7) return fail(IT_ERR_UNSUPPORTED_SHAPE, "widths must be multiples of 8, got %d", width);
    end += width;
    if (end > out_dim) break;
    p.out.end[r] = static_cast<int>(end);
    p.out.ptr[r] = r < n_outs ? outs[r] : nullptr;
    if (width > 0 && n > 0) {
      if (outs[r] == nullptr) return fail(IT_ERR_INVALID_ARG, "null tensor");
      if (!aligned16(outs[r])) return fail(IT_ERR_ALIGNMENT, "results must be 16-byte aligned");
    }
  }
  if (end != out_dim) return fail(IT_ERR_INVALID_ARG, "widths must add up to out_dim = %d", out_dim);
  if (n == 0 || out_dim == 0) return IT_OK;
  if (x_codes == nullptr || x_scales == nullptr || w_codes == nullptr || w_scales == nullptr) return fail(IT_ERR_INVALID_ARG, "null tensor");
  if (!aligned16(x_codes) || !aligned16(w_codes) || !aligned16(w_scales))
    return fail(IT_ERR_ALIGNMENT, "codes and weight scales must be 16-byte aligned");
  IT_CUDA(cudaSetDevice(ctx->device));
  p.x = x_codes;
  p.w = w_codes;
  p.sx = x_scales;
  p.sw = w_scales;
  p.M = n;
  p.N = out_dim;
  p.K = in_dim;
  p.status = ctx->d_status;
  return out_dtype == IT_F32 ? launch_linear_i8<float>(ctx, stream->s, p) : launch_linear_i8<__nv_bfloat16>(ctx, stream->s, p);
}
