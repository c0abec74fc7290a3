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

// x [rows, cols] -> codes [rows, cols], scales [rows].  A CTA per row, which keeps what it can of the row in registers between
// finding the largest magnitude and dividing: 8 columns a thread and step.
template <typename ST>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const ST* __restrict__ x, int8_t* __restrict__ codes, float* __restrict__ scales, int cols) {
  constexpr int KEEP = 4;
  __shared__ uint32_t s_most[8];
  const size_t row = blockIdx.x;
  const ST* src = x + row * cols;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  float keep[KEEP][8];
  uint32_t most = 0;
#pragma unroll
  for (int u = 0; u < KEEP; ++u) {
    const int c = (u * 256 + static_cast<int>(threadIdx.x)) * 8;
    if (c < cols) {
      q4_load8(src + c, keep[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(keep[u][e]) & 0x7FFFFFFFu);
    }
  }
  for (int c = (KEEP * 256 + static_cast<int>(threadIdx.x)) * 8; c < cols; c += 2048) {
    float v[8];
    q4_load8(src + c, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(v[e]) & 0x7FFFFFFFu);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) most = max(most, s_most[w]);
  const float s = quant_scale<127, 8>(most);
  const bool some = s > 0.f;
  const float inv = some ? __frcp_rn(s) : 0.f;
  if (threadIdx.x == 0) scales[row] = s;
  auto store = [&](int c, const float (&v)[8]) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e >> 2] |= (static_cast<uint32_t>(some ? quant_code<127>(v[e], s, inv) : 0) & 0xFFu) << (8 * (e & 3));
    *reinterpret_cast<uint2*>(codes + row * cols + c) = make_uint2(w[0], w[1]);
  };
#pragma unroll
  for (int u = 0; u < KEEP; ++u) {
    const int c = (u * 256 + static_cast<int>(threadIdx.x)) * 8;
    if (c < cols) store(c, keep[u]);
  }
  for (int c = (KEEP * 256 + static_cast<int>(threadIdx.x)) * 8; c < cols; c += 2048) {
    float v[8];
    q4_load8(src + c, v);
    store(c, v);
  }
}

// Where the columns of the product go: up to three column ranges, each a tensor [n, width] of its own.
struct I8Out {
  void* ptr[3];
  int end[3];      // first column behind the range
  int is_f32;
};
struct GemmI8Params {
  const float *sx, *sw;
  I8Out out;
  int M, N, K;
  int* status;
};

// 8 columns from `col` (a multiple of 8, as are the ranges' ends) of row `row`.
__device__ __forceinline__ void i8_store8(const I8Out& o, size_t row, int col, const float (&y)[8]) {
  const int r = col < o.end[0] ? 0 : col < o.end[1] ? 1 : 2;
  const int begin = r == 0 ? 0 : o.end[r - 1];
  const size_t at = row * (o.end[r] - begin) + (col - begin);
  if (o.is_f32) q4_store8(static_cast<float*>(o.ptr[r]) + at, y);
  else q4_store8(static_cast<__nv_bfloat16*>(o.ptr[r]) + at, y);
}

// The pipeline of gemm_bf16_sm100_kernel (y = x W^T) on bytes: a 128-byte row of a stage is 128 columns of K, an instruction of
// kind::i8 takes 32 of them, and tensor memory holds 32-bit integers.  Persistent CTAs (or pairs, CG = 2) of
//   warp 0: TMA loads   warp 1: tcgen05.mma   warp 2: tensor memory   warps 4-7: epilogue, a thread per row.
template <int BN, int CG>
__global__ void __launch_bounds__(256, 1)
gemm_i8_sm100_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const GemmI8Params prm) {
  using T = GemmTraits<BN, CG>;
  using namespace ptx;
  constexpr int BK = 128;   // bytes
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
      mbar_init(&acc_empty[i], CG == 2 ? 8 : 128);
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
      prefetch_tensormap(&tmap_a);
      prefetch_tensormap(&tmap_b);
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
            tma_load_4d_2cta(sa, &tmap_a, bar, kb * BK, m0, 0, 0);
            tma_load_4d_2cta(sb, &tmap_b, bar, kb * BK, n0, 0, 0);
          } else {
            mbar_arrive_expect_tx(&full[st], T::STAGE_BYTES);
            tma_load_4d(sa, &tmap_a, &full[st], kb * BK, m0, 0, 0);
            tma_load_4d(sb, &tmap_b, &full[st], kb * BK, n0, 0, 0);
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
    const int row_in_tile = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    int t = 0;
    bool ok = true;
    uint32_t r[32];
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
#pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        tmem_ld_x32(t_lane + buf * BN + c * 32, r);
        tmem_wait_ld();
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int col = n0 + c * 32 + v * 8;
          if (row < prm.M && col < prm.N) {
            float y[8], sw[8];
            q4_load8(prm.sw + col, sw);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = static_cast<float>(static_cast<int>(r[v * 8 + e])) * (sx * sw[e]);
            i8_store8(prm.out, row, col, y);
          }
        }
      }
      tc_fence_before();
      if (CG == 2) {
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(cluster_addr(&acc_empty[buf], 0));
      } else {
        mbar_arrive(&acc_empty[buf]);
      }
    }
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

}  // namespace it
