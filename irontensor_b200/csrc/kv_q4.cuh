// A key/value cache held in 4 bits: its form, writing new tokens into it, reading it back.
//
// 32 neighbouring columns of a head share a scale s; a value is s * c with a whole number c in -7..7:
//   s = (largest magnitude of the 32) / 7, rounded to 5 significant bits,     c = round(x / s), ties to even.
// 5 bits, because then s * c has at most 8 and is exact in bf16: attention's matrix instructions work on the very values that are
// read back, and the only error of the form is that of c.  A scale that is rounded down by its most, 1/33, leaves the largest
// magnitude at 7.22 steps, which is still 7.  Groups whose largest magnitude is below 2^-100 are zeros, one of more than
// 7 * 2^122 saturates, and one that holds a NaN or an infinity reads back as NaN.
//
// Row (one position of one K/V head) of head_dim columns, groups = ceil(head_dim / 32):
//   codes   4 * groups words of 32 bits; word t * groups + j holds columns 32 j + 8 t + e, e = 0..7, as c + 8 in the 4 bits from
//           4 * (e / 2) + 16 * (e % 2).  (Lane t of a quad takes `groups` consecutive words, one of each group, which is what
//           an operand fragment of mma.m16n8k16 is made of; two neighbouring columns come out of one mask as a register.)
//   scales  `groups` bf16
// Codes are [batch, kv_heads, max_len, 16 * groups] bytes and scales [batch, kv_heads, max_len, groups], for keys and values each:
// positions of a head follow one another, so a stretch of them is one contiguous piece.
#pragma once
#include <cuda_bf16.h>

#include <cfloat>
#include <cstdint>

#include "sm100_ptx.cuh"

namespace it {

// largest / MOST rounded to BITS significant bits, ties to even; NaN for a NaN or infinite `largest`, given by the bits of its
// magnitude.  The fp32 quotient is right but where it is rounded onto the middle between two results: there the sign of the
// remainder largest - MOST * quotient, exact in one fma, decides.
template <int MOST, int BITS>
__device__ __forceinline__ float quant_scale(uint32_t largest_bits) {
  if (largest_bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  const float largest = __uint_as_float(largest_bits);
  if (largest < 0x1p-100f) return 0.f;
  constexpr int DROP = 24 - BITS;
  constexpr uint32_t MASK = (1u << DROP) - 1u, HALF = 1u << (DROP - 1);
  const float t = __fdiv_rn(largest, static_cast<float>(MOST));
  const float rest = fmaf(-static_cast<float>(MOST), t, largest);
  const uint32_t bits = __float_as_uint(t), low = bits & MASK, base = bits & ~MASK;
  const bool up = low > HALF || (low == HALF && (rest > 0.f || (rest == 0.f && ((base >> DROP) & 1u))));
  return __uint_as_float(base + (up ? MASK + 1u : 0u));
}

// round(x / s), ties to even, for s of at most 8 significant bits; inv = 1 / s.  x * inv may be a step off next to the middle of
// two whole numbers; x - q s is exact there (at most 24 bits above the last place of x) and says which is nearer.
template <int MOST>
__device__ __forceinline__ int quant_code(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = fmaf(-q, s, x), half = 0.5f * s;
  const bool odd = static_cast<int>(q) & 1;
  if (r > half || (r == half && odd)) q += 1.f;
  else if (r < -half || (r == -half && odd)) q -= 1.f;
  return static_cast<int>(fminf(fmaxf(q, -static_cast<float>(MOST)), static_cast<float>(MOST)));
}

constexpr float Q4_MOST_SCALE = 0x1p122f;   // 24 * s, which attention's operands are made with, stays finite

struct KvQ4 {   // one of the two halves of a cache
  uint32_t* codes;          // words
  __nv_bfloat16* scales;
};

__device__ __forceinline__ void q4_load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void q4_load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void q4_store8(__nv_bfloat16* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(ptx::pack_bf16(x[0], x[1]), ptx::pack_bf16(x[2], x[3]), ptx::pack_bf16(x[4], x[5]),
                                            ptx::pack_bf16(x[6], x[7]));
}
__device__ __forceinline__ void q4_store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

// New tokens k, v [batch, T, kv_heads, head_dim] into the cache behind the lengths[b] positions that are there; of sequence b the
// first counts[b] tokens (null: all T).  new_lengths[b] = what is there afterwards.  A thread takes 8 columns, the quad that shares
// a group finds its largest magnitude by two shuffles.  Positions outside the cache are not written, and reported.
// Reads 2 * 8 or 4 * 8 bytes a thread and writes 4.5: bound by memory, and for single tokens by the launch.
template <typename ST>
__global__ void __launch_bounds__(256)
kv_q4_append_kernel(const ST* __restrict__ k, const ST* __restrict__ v, KvQ4 ck, KvQ4 cv, const int* __restrict__ lengths,
                    const int* __restrict__ counts, int* __restrict__ new_lengths, int B, int T, int Hkv, int D, int max_len, int* status) {
  const int groups = (D + 31) >> 5, lanes = 4 * groups;   // threads of a row
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const long long rows = static_cast<long long>(B) * T * Hkv, total = 2 * rows * lanes;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i < B) {
    const int have = lengths[i], want = counts != nullptr ? counts[i] : T, add = min(max(want, 0), T);
    const long long end = static_cast<long long>(have) + add;
    if (have < 0 || end > max_len || add != want) atomicCAS(status, 0, DEV_ERR_CACHE_RANGE);
    new_lengths[i] = static_cast<int>(min(max(end, 0LL), static_cast<long long>(max_len)));
  }
  const bool live = i < total;   // a quad is live as a whole; its warp stays together for the shuffles
  const long long at = live ? i : 0;
  const bool is_v = at >= rows * lanes;
  const long long in_half = is_v ? at - rows * lanes : at;
  const long long row = in_half / lanes;
  const int lane = static_cast<int>(in_half - row * lanes), j = lane >> 2, t = lane & 3;
  const int h = static_cast<int>(row % Hkv);
  const long long bt = row / Hkv;
  const int b = static_cast<int>(bt / T), tok = static_cast<int>(bt - static_cast<long long>(b) * T);
  const int d0 = 32 * j + 8 * t;
  float x[8] = {};
  if (live && d0 < D) q4_load8((is_v ? v : k) + row * D + d0, x);
  uint32_t largest = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) largest = max(largest, __float_as_uint(x[e]) & 0x7FFFFFFFu);
  largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
  largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
  float s = quant_scale<7, 5>(largest);
  if (s > Q4_MOST_SCALE) s = Q4_MOST_SCALE;
  const bool some = s > 0.f;   // false for NaN too
  const float inv = some ? __frcp_rn(s) : 0.f;
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = some ? quant_code<7>(x[e], s, inv) : 0;
    word |= static_cast<uint32_t>(c + 8) << (4 * (e >> 1) + 16 * (e & 1));
  }
  if (!live || tok >= (counts != nullptr ? counts[b] : T)) return;
  const long long pos = static_cast<long long>(lengths[b]) + tok;
  if (pos < 0 || pos >= max_len) return;
  const long long crow = (static_cast<long long>(b) * Hkv + h) * max_len + pos;
  const KvQ4& c = is_v ? cv : ck;
  c.codes[crow * lanes + t * groups + j] = word;
  if (t == 0) c.scales[crow * groups + j] = __float2bfloat16_rn(s);
}

// Positions starts[b] + t, t < T, of the cache (null: from 0) as keys and values [batch, T, kv_heads, head_dim]; zeros outside
// 0 <= position < min(lengths[b], max_len) (null: max_len).  A thread writes 8 columns.  Bound by the bytes that it writes.
template <typename ST>
__global__ void __launch_bounds__(256)
kv_q4_read_kernel(ST* __restrict__ k, ST* __restrict__ v, KvQ4 ck, KvQ4 cv, const int* __restrict__ starts, const int* __restrict__ lengths,
                  int B, int T, int Hkv, int D, int max_len) {
  const int groups = (D + 31) >> 5, per_row = D >> 3;   // threads of a row: none for a padded group's empty columns
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const long long rows = static_cast<long long>(B) * T * Hkv, total = 2 * rows * per_row;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const bool is_v = i >= rows * per_row;
  const long long in_half = is_v ? i - rows * per_row : i;
  const long long row = in_half / per_row;
  const int oct = static_cast<int>(in_half - row * per_row), j = oct >> 2, t = oct & 3;
  const int h = static_cast<int>(row % Hkv);
  const long long bt = row / Hkv;
  const int b = static_cast<int>(bt / T), tok = static_cast<int>(bt - static_cast<long long>(b) * T);
  const long long pos = static_cast<long long>(starts != nullptr ? starts[b] : 0) + tok;
  const int end = lengths != nullptr ? min(lengths[b], max_len) : max_len;
  float x[8] = {};
  if (pos >= 0 && pos < end) {
    const long long crow = (static_cast<long long>(b) * Hkv + h) * max_len + pos;
    const KvQ4& c = is_v ? cv : ck;
    const uint32_t w = __ldg(c.codes + crow * 4 * groups + t * groups + j);
    const float s = __bfloat162float(c.scales[crow * groups + j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = s * static_cast<float>(static_cast<int>((w >> (4 * (e >> 1) + 16 * (e & 1))) & 15u) - 8);
  }
  q4_store8((is_v ? v : k) + row * D + 8 * oct, x);
}

}  // namespace it
