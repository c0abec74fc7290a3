// Projections in 8-bit integers: y[n, out] = (cx cw^T)[n, out] * sx[n] * sw[out], with tokens cx, sx quantised row by row and weights
// cw, sw channel by channel.
//
// A row's scale is (its largest magnitude / 127) rounded to 8 significant bits, a value is scale * c with a whole number c in
// -127..127 (quant_scale, quant_code in kv_q4.cuh).  8 bits, so that every decision between two whole numbers is exact in fp32 and so
// is the product of two scales.  Sums of products are 32-bit integers and exact; the result is rounded where they become fp32
// (2^-24), where the scales' product is applied (2^-24) and where it is stored.
#pragma once
#include <cuda_bf16.h>

#include <cstdint>

#include "gemm_sm100.cuh"
#include "kv_q4.cuh"
#include "sm100_ptx.cuh"

namespace it {

// x [rows, cols] -> codes [rows, cols], scales [rows].  WARPS warps a row, which keep what they can of it (16 bytes a lane and step,
// KEEP steps) in registers between finding the largest magnitude and dividing, and read the rest again.  Bound by memory where
// there are many rows, and by two trips to it where there are few.
template <typename ST, int WARPS>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const ST* __restrict__ x, int8_t* __restrict__ codes, float* __restrict__ scales, int rows, int cols) {
  constexpr int KEEP = 8, VEC = 16 / sizeof(ST), STEP = 32 * WARPS * VEC, ROWS = 8 / WARPS;
  __shared__ uint32_t s_most[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * ROWS + warp / WARPS;
  const int first = ((warp % WARPS) * 32 + lane) * VEC;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  if (WARPS == 1 && row >= rows) return;   // a row of more warps is a whole CTA's, or half of one: all stay for the barrier
  const ST* src = x + (row < rows ? row : 0) * cols;
  auto bits = [](const uint4& v, uint32_t most) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(ST) == 4) most = max(most, w[i] & 0x7FFFFFFFu);
      else most = max(most, max((w[i] << 16) & 0x7FFFFFFFu, w[i] & 0x7FFF0000u));
    }
    return most;
  };
  uint4 keep[KEEP];
  uint32_t most = 0;
#pragma unroll
  for (int u = 0; u < KEEP; ++u) {
    keep[u] = make_uint4(0u, 0u, 0u, 0u);
    if (first + u * STEP < cols) keep[u] = __ldg(reinterpret_cast<const uint4*>(src + first + u * STEP));
  }
#pragma unroll
  for (int u = 0; u < KEEP; ++u) most = bits(keep[u], most);
  for (int c = first + KEEP * STEP; c < cols; c += STEP) most = bits(__ldg(reinterpret_cast<const uint4*>(src + c)), most);
  most = __reduce_max_sync(0xffffffffu, most);
  if (WARPS > 1) {
    if (lane == 0) s_most[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) most = max(most, s_most[warp / WARPS * WARPS + w]);
    if (row >= rows) return;
  }
  const float s = quant_scale<127, 8>(most);
  const bool some = s > 0.f;   // false: zeros, or not numbers
  const float inv = quant_inverse(s);
  if (first == 0) scales[row] = s;
  auto store = [&](int c, const uint4& v) {
    float f[VEC];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(ST) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
    uint32_t b[VEC] = {};
    if (some) quant_codes<0, sizeof(ST) == 2>(f, s, inv, b);
    uint32_t out[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      out[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(codes + row * cols + c) = make_uint2(out[0], out[1]);
    else *reinterpret_cast<uint32_t*>(codes + row * cols + c) = out[0];
  };
#pragma unroll
  for (int u = 0; u < KEEP; ++u)
    if (first + u * STEP < cols) store(first + u * STEP, keep[u]);
  for (int c = first + KEEP * STEP; c < cols; c += STEP) store(c, __ldg(reinterpret_cast<const uint4*>(src + c)));
}

// Where the columns of the product go: up to three column ranges, each a tensor [n, width] of its own.
struct I8Out {
  void* ptr[3];
  int end[3];      // first column behind the range
};
struct GemmI8Params {
  const int8_t *x, *w;
  const float *sx, *sw;
  I8Out out;
  int M, N, K;
  int* status;
};
struct GemmI8Maps {   // x and w as bytes, and the results: boxes of 128 bytes by 32 rows, 128-byte swizzle
  CUtensorMap a, b, out[3];
};

__device__ __forceinline__ int i8_range_of(const I8Out& o, int col) { return col < o.end[0] ? 0 : col < o.end[1] ? 1 : 2; }
__device__ __forceinline__ int i8_range_begin(const I8Out& o, int r) { return r == 0 ? 0 : o.end[r - 1]; }
// 8 columns from `col` (a multiple of 8, as are the ranges' ends) of row `row`.
template <typename OT>
__device__ __forceinline__ void i8_store8(const I8Out& o, size_t row, int col, const float (&y)[8]) {
  const int r = i8_range_of(o, col), begin = i8_range_begin(o, r);
  q4_store8(static_cast<OT*>(o.ptr[r]) + row * (o.end[r] - begin) + (col - begin), y);
}

template <int BN_, int CG>
struct GemmI8Traits {
  static constexpr int BM = 128, BK = 128, B_ROWS = BN_ / CG;
  static constexpr int A_BYTES = BM * BK, B_BYTES = B_ROWS * BK, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = B_ROWS == 256 ? 4 : B_ROWS == 128 ? 6 : 8;
  static constexpr int OUT_BYTES = 32 * 128;                  // a warp's piece of the result
  static constexpr int OUT_WARPS = 8;
  static constexpr int SMEM_OUT = STAGES * STAGE_BYTES;
  static constexpr int SMEM_BAR = SMEM_OUT + OUT_WARPS * OUT_BYTES;
  static constexpr int SMEM_MISC = SMEM_BAR + (2 * STAGES + 4) * 8;
  static constexpr int SMEM_BYTES = SMEM_MISC + 16;
  static constexpr int THREADS = 128 + 32 * OUT_WARPS;
  static constexpr uint32_t TMEM_COLS = 2 * BN_;              // two accumulators
};

// The pipeline of gemm_bf16_sm100_kernel (y = x W^T) on bytes: a 128-byte row of a stage is 128 columns of K, an instruction of
// kind::i8 takes 32 of them, and tensor memory holds 32-bit integers.  Persistent CTAs (or pairs, CG = 2) of
//   warp 0: TMA loads   warp 1: tcgen05.mma   warp 2: tensor memory   warps 4-11: epilogue, two warps for 32 rows.
// At twice bf16's rate a tile has half the time for its epilogue.  Stored from registers, 16 bytes of 32 rows at a time, results of
// 2999 x 2048 -> 6144 took 71 us in fp32; so a warp turns pieces of 32 rows by 128 bytes round in shared memory and stores them
// by TMA: whole lines, and no instructions of the epilogue's (2999 x 2048 by 6144, fp32: 71 -> 35 us).
template <int BN, int CG, typename OT>
__global__ void __launch_bounds__(384, 1)
gemm_i8_sm100_kernel(const __grid_constant__ GemmI8Maps maps, const GemmI8Params prm) {
  using T = GemmI8Traits<BN, CG>;
  using namespace ptx;
  constexpr int BK = T::BK;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + T::SMEM_BAR);
  uint64_t* full = bars;
  uint64_t* empty = full + T::STAGES;
  uint64_t* acc_full = empty + T::STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + T::SMEM_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + T::SMEM_MISC + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? static_cast<int>(blockIdx.x) & 1 : 0;
  const int first_tile = static_cast<int>(blockIdx.x) / CG, tile_step = static_cast<int>(gridDim.x) / CG;
  const int tiles_m = (prm.M + CG * T::BM - 1) / (CG * T::BM), tiles_n = (prm.N + BN - 1) / BN;
  const int n_tiles = tiles_m * tiles_n;
  const int n_kb = (prm.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    if (smem_addr(smem) & 1023u) {
      *abort_flag = 1;
      atomicCAS(prm.status, 0, DEV_ERR_SMEM_ALIGN);
    }
    if (*reinterpret_cast<volatile int*>(prm.status) != 0) *abort_flag = 1;
    for (int i = 0; i < T::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], CG * T::OUT_WARPS);   // one arrival per epilogue warp, of a pair of both CTAs
    }
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 2) {
    if (CG == 2) {
      tmem_alloc_2cta(tmem_slot, T::TMEM_COLS);
      tmem_relinquish_2cta();
    } else {
      tmem_alloc(tmem_slot, T::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();
  tc_fence_after();
  grid_dep_wait();
  grid_dep_launch();
  const uint32_t tmem_base = *tmem_slot;
  const bool run = *abort_flag == 0;

  if (!run) {
    // nothing to do
  } else if (warp == 0) {
    if (elect_one()) {
      prefetch_tensormap(&maps.a);
      prefetch_tensormap(&maps.b);
      int it = 0;
      bool ok = true;
      for (int tile = first_tile; tile < n_tiles && ok; tile += tile_step) {
        int tm, tn;
        gemm_tile_coords(tile, tiles_m, tiles_n, &tm, &tn);
        const int m0 = (tm * CG + rank) * T::BM, n0 = tn * BN + rank * T::B_ROWS;
        for (int kb = 0; kb < n_kb; ++kb, ++it) {
          const int st = it % T::STAGES;
          ok = mbar_wait(&empty[st], ((it / T::STAGES) & 1) ^ 1, abort_flag, prm.status, DEV_ERR_TIMEOUT_EMPTY);
          if (!ok) break;
          uint8_t* sa = smem + st * T::STAGE_BYTES;
          uint8_t* sb = sa + T::A_BYTES;
          if (CG == 2) {   // the even CTA expects both CTAs' bytes
            if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * T::STAGE_BYTES);
            const uint32_t bar = cluster_addr(&full[st], 0);
            tma_load_4d_2cta(sa, &maps.a, bar, kb * BK, m0, 0, 0);
            tma_load_4d_2cta(sb, &maps.b, bar, kb * BK, n0, 0, 0);
          } else {
            mbar_arrive_expect_tx(&full[st], T::STAGE_BYTES);
            tma_load_4d(sa, &maps.a, &full[st], kb * BK, m0, 0, 0);
            tma_load_4d(sb, &maps.b, &full[st], kb * BK, n0, 0, 0);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t IDESC = make_idesc_i8(CG * T::BM, BN);
      int it = 0, t = 0;
      bool ok = true;
      for (int tile = first_tile; tile < n_tiles && ok; tile += tile_step, ++t) {
        const int buf = t & 1;
        ok = mbar_wait(&acc_empty[buf], ((t >> 1) & 1) ^ 1, abort_flag, prm.status, DEV_ERR_TIMEOUT_SOFTMAX);
        if (!ok) break;
        tc_fence_after();
        for (int kb = 0; kb < n_kb; ++kb, ++it) {
          const int st = it % T::STAGES;
          ok = mbar_wait(&full[st], (it / T::STAGES) & 1, abort_flag, prm.status, DEV_ERR_TIMEOUT_LOAD);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_addr = smem_addr(smem + st * T::STAGE_BYTES);
          const uint64_t da = make_sdesc(a_addr, 16, 1024), db = make_sdesc(a_addr + T::A_BYTES, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t accumulate = (kb > 0 || kk > 0) ? 1u : 0u;
            if (CG == 2)
              umma_i8_ss_2cta(tmem_base + buf * BN, sdesc_advance(da, kk * 32), sdesc_advance(db, kk * 32), IDESC, accumulate);
            else
              umma_i8_ss(tmem_base + buf * BN, sdesc_advance(da, kk * 32), sdesc_advance(db, kk * 32), IDESC, accumulate);
          }
          if (CG == 2)
            umma_commit_2cta(&empty[st]);
          else
            umma_commit(&empty[st]);
        }
        if (ok) {
          if (CG == 2)
            umma_commit_2cta(&acc_full[buf]);
          else
            umma_commit(&acc_full[buf]);
        }
      }
    }
  } else if (warp >= 4) {
    constexpr int W = 128 / sizeof(OT);      // columns of a piece
    const int row_in_tile = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    uint8_t* piece = smem + T::SMEM_OUT + (warp - 4) * T::OUT_BYTES;
    int t = 0;
    bool ok = true;
    for (int tile = first_tile; tile < n_tiles && ok; tile += tile_step, ++t) {
      const int buf = t & 1;
      int tm, tn;
      gemm_tile_coords(tile, tiles_m, tiles_n, &tm, &tn);
      const int m0 = (tm * CG + rank) * T::BM, n0 = tn * BN, row = m0 + row_in_tile;
      const float sx = row < prm.M ? prm.sx[row] : 0.f;
      ok = mbar_wait(&acc_full[buf], (t >> 1) & 1, abort_flag, prm.status, DEV_ERR_TIMEOUT_MMA);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      if (m0 + (warp & 3) * 32 < prm.M) {
#pragma unroll 1
        for (int c = (warp - 4) >> 2; c < BN / W; c += 2) {
          const int col0 = n0 + c * W;
          if (col0 >= prm.N) break;
          // a piece that lies in one range (what is behind the range's last column is cut off) goes through shared memory
          const int range = i8_range_of(prm.out, col0), begin = i8_range_begin(prm.out, range);
          const bool whole = min(col0 + W, prm.N) <= prm.out.end[range];
          uint32_t out[32];   // the row's 128 bytes
#pragma unroll
          for (int half = 0; half < W / 32; ++half) {
            uint32_t r[32];
            tmem_ld_x32(t_lane + buf * BN + c * W + half * 32, r);
            float4 sw[8];
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              const int col = col0 + half * 32 + v * 4;
              sw[v] = col < prm.N ? __ldg(reinterpret_cast<const float4*>(prm.sw + col)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            tmem_wait_ld();
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const float f[8] = {sw[2 * v].x, sw[2 * v].y, sw[2 * v].z, sw[2 * v].w, sw[2 * v + 1].x, sw[2 * v + 1].y, sw[2 * v + 1].z, sw[2 * v + 1].w};
              float y[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = static_cast<float>(static_cast<int>(r[v * 8 + e])) * (sx * f[e]);
              if (!whole) {
                const int col = col0 + half * 32 + v * 8;
                if (row < prm.M && col < prm.N) i8_store8<OT>(prm.out, row, col, y);
              }
              if constexpr (sizeof(OT) == 4) {
#pragma unroll
                for (int e = 0; e < 8; ++e) out[v * 8 + e] = __float_as_uint(y[e]);
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) out[half * 16 + v * 4 + e] = pack_bf16(y[2 * e], y[2 * e + 1]);
              }
            }
          }
          if (whole) {
            if (lane == 0) bulk_wait_group_read<0>();   // the piece before has left the buffer
            __syncwarp();
#pragma unroll
            for (int v = 0; v < 8; ++v)
              *reinterpret_cast<uint4*>(piece + lane * 128 + ((v ^ (lane & 7)) << 4)) = make_uint4(out[4 * v], out[4 * v + 1], out[4 * v + 2], out[4 * v + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_4d(&maps.out[range], piece, col0 - begin, m0 + (warp & 3) * 32, 0, 0);
              bulk_commit_group();
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2) mbar_arrive_cluster(cluster_addr(&acc_empty[buf], 0));
        else mbar_arrive(&acc_empty[buf]);
      }
    }
    if (lane == 0) bulk_wait_group_all();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  // a CTA that gave up lets what it has in flight land before its memory goes away
  if (*abort_flag)
    for (int i = 0; i < 50; ++i) __nanosleep(20000);
  if (CG == 2) {
    __syncwarp();
    cluster_sync_all();
    if (warp == 2) {
      tc_fence_after();
      tmem_dealloc_2cta(tmem_base, T::TMEM_COLS);
    }
  } else if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, T::TMEM_COLS);
  }
}

__device__ __forceinline__ void mma_s8_16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A handful of tokens: every SM streams weights, as gemm_skinny_kernel does for bf16 and for the same reason.  A CTA owns 16 channels,
// its eight warps split K, a lane reads 16 bytes of a row at a time; the four lanes of a quad hold 64 consecutive k, in the same
// order for channels and tokens.  NT: groups of 8 tokens.
template <int NT, typename OT>
__global__ void __launch_bounds__(256)
gemm_i8_skinny_kernel(const GemmI8Params p) {
  constexpr int WARPS = 8, U = NT <= 2 ? 4 : 2, TOK = NT * 8, ROWS = 16;
  __shared__ int part[WARPS][ROWS][TOK + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int r0 = blockIdx.x * ROWS;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  int acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0;
  const int steps = (p.K + 63) >> 6;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int s0 = warp * U; s0 < steps; s0 += WARPS * U) {
    uint4 a[U][2], b[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (s0 + u) * 64 + t * 16;
      const bool ok = k < p.K;    // K is a multiple of 16
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = r0 + h * 8 + g;
        a[u][h] = (ok && row < p.N) ? __ldg(reinterpret_cast<const uint4*>(p.w + static_cast<size_t>(row) * p.K + k)) : zero;
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int tok = j * 8 + g;
        b[u][j] = (ok && tok < p.M) ? *reinterpret_cast<const uint4*>(p.x + static_cast<size_t>(tok) * p.K + k) : zero;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma_s8_16832(acc[j], a[u][0].x, a[u][1].x, a[u][0].y, a[u][1].y, b[u][j].x, b[u][j].y);
        mma_s8_16832(acc[j], a[u][0].z, a[u][1].z, a[u][0].w, a[u][1].w, b[u][j].z, b[u][j].w);
      }
  }
  // c0, c1: row g, tokens 2t, 2t + 1; c2, c3: row g + 8
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[warp][(e >> 1) * 8 + g][j * 8 + t * 2 + (e & 1)] = acc[j][e];
  __syncthreads();
  // a thread finishes pairs of neighbouring columns of y, which lie in one range
  for (int idx = threadIdx.x; idx < TOK * (ROWS / 2); idx += 256) {
    const int tok = idx / (ROWS / 2), pr = idx - tok * (ROWS / 2);
    const int col = r0 + 2 * pr;
    if (tok >= p.M || col >= p.N) continue;
    int v0 = 0, v1 = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      v0 += part[w][2 * pr][tok];
      v1 += part[w][2 * pr + 1][tok];
    }
    const float sx = p.sx[tok], y0 = static_cast<float>(v0) * (sx * p.sw[col]), y1 = static_cast<float>(v1) * (sx * p.sw[col + 1]);
    const int r = i8_range_of(p.out, col), begin = i8_range_begin(p.out, r);
    OT* dst = static_cast<OT*>(p.out.ptr[r]) + static_cast<size_t>(tok) * (p.out.end[r] - begin) + (col - begin);
    if constexpr (sizeof(OT) == 4) *reinterpret_cast<float2*>(dst) = make_float2(y0, y1);
    else *reinterpret_cast<uint32_t*>(dst) = ptx::pack_bf16(y0, y1);
  }
}

}  // namespace it
