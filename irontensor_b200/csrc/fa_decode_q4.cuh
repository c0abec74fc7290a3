// Attention for one new token per sequence against a 4-bit key/value cache (kv_q4.cuh), every sequence at its own length:
// o[b, h] = softmax(q[b, h] K^T / sqrt(D)) V over the first lengths[b] positions of K/V head h / (heads / kv_heads).
//
// A value of the cache is c * s, exact in bf16.  A nibble u = c + 8 masked into the upper mantissa bits of a bf16 whose exponent
// says 16 is the number 16 + u, and (16 + u) * s - 24 * s = c * s is one fma of two packed values, exact because 24 * s has 7
// significant bits and c * s at most 8.  So a 32-bit word of eight codes becomes four operand registers by a shift, a mask and an
// fma each, and everything behind that is bf16 matrix instructions (mma.sync m16n8k16, fp32 sums):
//   S = Q K^T   rows: up to 8 query heads; B: 8 keys by 16 columns, which lie together in a word of the cache
//   O = P V     rows: the same heads; B: 16 keys by 8 columns.  A register holds one column of two keys, so two keys' words are
//               interleaved by halves first (two byte permutes for 16 codes).
// Eight heads fill half of the 16 rows.  The other half carries the next bits of the same heads' operand: P goes in as the two
// bf16 terms hi (rows 0-7) and lo (rows 8-15), 16 bits in one instruction, and the two halves of the result are added at the end;
// an fp32 q likewise, with a third term in an instruction of its own, as has its P.
// Which key is which column of S, and which column of V is which column of O, is free as long as both products agree: the order
// is the one in which the words lie (dims_of).
//
// A warp walks blocks of 32 keys with an online softmax of its own; warps merge through shared memory, and the ranges of keys
// that a launch splits a sequence into (even shares of lengths[b], which only the device knows) through a second launch.
#pragma once
#include <cuda_bf16.h>

#include <cstdint>

#include "gemm_skinny.cuh"
#include "kv_q4.cuh"
#include "sm100_ptx.cuh"

namespace it {

constexpr int DQ_WARPS = 8, DQ_BLOCK = 32, DQ_HEADS = 8, DQ_MAX_SPLITS = 64;

struct DecodeQ4Params {
  const void* q;            // [batch, heads, D]
  const uint32_t *k_codes, *v_codes;
  const __nv_bfloat16 *k_scales, *v_scales;
  const int* lengths;
  void* o;
  float *lse, *part_o, *part_ml;
  int* status;
  int H, Hkv, D, max_len, n_splits;
  float scale_log2;         // 1/sqrt(D) * log2(e)
};

__device__ __forceinline__ uint32_t q4_fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t q4_mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Nibble I of both halves of w as the values (16 + u) s - 24 s.
template <int I>
__device__ __forceinline__ uint32_t q4_pair(uint32_t w, uint32_t s2, uint32_t bias2) {
  const uint32_t at3 = I == 0 ? w << 3 : w >> (4 * I - 3);
  return q4_fma2((at3 & 0x00780078u) | 0x41804180u, s2, bias2);
}
constexpr uint32_t Q4_MINUS_24 = 0xC1C0C1C0u;   // -24 in both halves

// Which column of a head is n-tile nt's column n of O (see the V operand below).
template <int NG>
__device__ __forceinline__ int q4_dim_of(int nt, int n) {
  constexpr int F = NG / 2;
  int w, e;
  if (nt < 8 * F) {
    w = n * F + nt / 8;                  // whole sets of 8 words: lane n owns F consecutive words
    e = nt % 8;
  } else {
    w = 8 * F + (n & 3);                 // the last 4 words, of which lanes 4-7 take the odd columns
    e = 2 * (nt - 8 * F) + (n >> 2);
  }
  return 32 * (w % NG) + 8 * (w / NG) + e;
}

// NG: groups of 32 columns; TERMS: bf16 terms of q and P (1: bf16 q, two-term P; 3: fp32 q, three-term P).
template <int NG, int TERMS>
__global__ void __launch_bounds__(32 * DQ_WARPS, 1)
fa_decode_q4_kernel(const DecodeQ4Params prm) {
  using ST = typename std::conditional<TERMS == 1, __nv_bfloat16, float>::type;
  constexpr int NT = 4 * NG, F = NG / 2, HALF = NG & 1;   // n-tiles of O; whole sets of 8 words; a set of 4
  __shared__ float s_acc[DQ_WARPS][DQ_HEADS][32 * NG];
  __shared__ float s_ml[DQ_WARPS][DQ_HEADS][2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = prm.H / prm.Hkv, chunks = (G + DQ_HEADS - 1) / DQ_HEADS;
  const int b = blockIdx.z, hk = static_cast<int>(blockIdx.y) / chunks, g0 = (static_cast<int>(blockIdx.y) % chunks) * DQ_HEADS;
  const int gc = min(DQ_HEADS, G - g0), sp = blockIdx.x, D = prm.D;
  const size_t bh0 = static_cast<size_t>(b) * prm.H + hk * G + g0;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int given = prm.lengths[b], len = min(max(given, 0), prm.max_len);
  if (given != len && threadIdx.x == 0) atomicCAS(prm.status, 0, DEV_ERR_CACHE_RANGE);
  const int blocks = (len + DQ_BLOCK - 1) / DQ_BLOCK, share = (blocks + prm.n_splits - 1) / prm.n_splits;
  const int k_begin = min(sp * share * DQ_BLOCK, len), k_end = min((sp + 1) * share * DQ_BLOCK, len);

  // q: register 4 j + r holds columns 32 j + 8 t + 2 r and the next, of head g; its further terms for fp32
  uint32_t qa[TERMS][4 * NG];
#pragma unroll
  for (int i = 0; i < 4 * NG; ++i) {
    const int d = 32 * (i >> 2) + 8 * t + 2 * (i & 3);
    float x0 = 0.f, x1 = 0.f;
    if (g < gc && d < D) {
      const ST* src = static_cast<const ST*>(prm.q) + (bh0 + g) * D + d;
      x0 = rope_ld(src);
      x1 = rope_ld(src + 1);
    }
#pragma unroll
    for (int n = 0; n < TERMS; ++n) {
      qa[n][i] = ptx::pack_bf16(x0, x1);
      x0 -= __uint_as_float(qa[n][i] << 16);
      x1 -= __uint_as_float(qa[n][i] & 0xFFFF0000u);
    }
  }
  float acc[NT][4], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;

  const size_t row0 = (static_cast<size_t>(b) * prm.Hkv + hk) * prm.max_len;
  for (int k0 = k_begin + warp * DQ_BLOCK; k0 < k_end; k0 += DQ_WARPS * DQ_BLOCK) {
    // ---- scores of 4 x 8 keys: lane g's key is the n index, lanes t share its columns
    float s[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const size_t row = row0 + min(k0 + 8 * i + g, k_end - 1);
      const uint32_t* src = prm.k_codes + row * (4 * NG) + t * NG;
      uint32_t w[NG];
#pragma unroll
      for (int j = 0; j < NG; ++j) w[j] = __ldg(src + j);
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t s1 = __ldg(reinterpret_cast<const unsigned short*>(prm.k_scales) + row * NG + j);
        const uint32_t s2 = __byte_perm(s1, 0, 0x1010), bias2 = q4_mul2(s2, Q4_MINUS_24);
        const uint32_t b0 = q4_pair<0>(w[j], s2, bias2), b1 = q4_pair<1>(w[j], s2, bias2);
        const uint32_t b2 = q4_pair<2>(w[j], s2, bias2), b3 = q4_pair<3>(w[j], s2, bias2);
        if constexpr (TERMS == 1) {
          mma_bf16_16816(c, qa[0][4 * j], 0u, qa[0][4 * j + 1], 0u, b0, b1);
          mma_bf16_16816(c, qa[0][4 * j + 2], 0u, qa[0][4 * j + 3], 0u, b2, b3);
        } else {
          mma_bf16_16816(c, qa[0][4 * j], qa[1][4 * j], qa[0][4 * j + 1], qa[1][4 * j + 1], b0, b1);
          mma_bf16_16816(c, qa[0][4 * j + 2], qa[1][4 * j + 2], qa[0][4 * j + 3], qa[1][4 * j + 3], b2, b3);
          mma_bf16_16816(c, 0u, qa[TERMS - 1][4 * j], 0u, qa[TERMS - 1][4 * j + 1], b0, b1);
          mma_bf16_16816(c, 0u, qa[TERMS - 1][4 * j + 2], 0u, qa[TERMS - 1][4 * j + 3], b2, b3);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[i][e] = TERMS == 1 ? c[e] : c[e] + c[e + 2];
        if (k0 + 8 * i + 2 * t + e >= k_end) s[i][e] = -INFINITY;
      }
    }
    // ---- online softmax of head g; a lane holds 8 of the 32 keys
    float mx = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaxf(s[i][0], s[i][1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float m_ref = mx == -INFINITY ? 0.f : mx * prm.scale_log2;
    if (__any_sync(0xffffffffu, mx > m)) {
      const float corr = ptx::ex2(fmaf(m, prm.scale_log2, -m_ref));
      l *= corr;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] *= corr;
      m = mx;
    }
    uint32_t hi[4], lo[4], third[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float p0 = ptx::ex2(fmaf(s[i][0], prm.scale_log2, -m_ref)), p1 = ptx::ex2(fmaf(s[i][1], prm.scale_log2, -m_ref));
      l += p0 + p1;
      hi[i] = ptx::pack_bf16(p0, p1);
      p0 -= __uint_as_float(hi[i] << 16);
      p1 -= __uint_as_float(hi[i] & 0xFFFF0000u);
      lo[i] = ptx::pack_bf16(p0, p1);
      if (TERMS > 1) third[i] = ptx::pack_bf16_rest(lo[i], p0, p1);
    }
    // ---- O += P V, 16 keys at a time: registers of keys (2t, 2t + 1) and (2t + 8, 2t + 9)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      size_t rows[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) rows[n] = row0 + min(k0 + 16 * h + 2 * t + (n & 1) + 8 * (n >> 1), k_end - 1);
      auto product = [&](int nt, uint32_t b0, uint32_t b1) {
        mma_bf16_16816(acc[nt], hi[2 * h], lo[2 * h], hi[2 * h + 1], lo[2 * h + 1], b0, b1);
        if (TERMS > 1) mma_bf16_16816(acc[nt], third[2 * h], 0u, third[2 * h + 1], 0u, b0, b1);
      };
#pragma unroll
      for (int f = 0; f < F + HALF; ++f) {
        const bool whole = f < F;
        const int word = whole ? g * F + f : 8 * F + (g & 3);
        uint32_t w[4], s2[2], bias2[2];
#pragma unroll
        for (int n = 0; n < 4; ++n) w[n] = __ldg(prm.v_codes + rows[n] * (4 * NG) + word);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const unsigned short* sc = reinterpret_cast<const unsigned short*>(prm.v_scales);
          s2[n] = __byte_perm(__ldg(sc + rows[2 * n] * NG + word % NG), __ldg(sc + rows[2 * n + 1] * NG + word % NG), 0x5410);
          bias2[n] = q4_mul2(s2[n], Q4_MINUS_24);
        }
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {   // the low halves of two keys' words: even columns; the high halves: odd ones
          if (!whole && odd == 1) break;
          const uint32_t sel = whole ? (odd ? 0x7632u : 0x5410u) : (g & 4 ? 0x7632u : 0x5410u);
          const uint32_t a = __byte_perm(w[0], w[1], sel), c = __byte_perm(w[2], w[3], sel);
          const int nt = whole ? 8 * f + odd : 8 * F, step = whole ? 2 : 1;
          product(nt, q4_pair<0>(a, s2[0], bias2[0]), q4_pair<0>(c, s2[1], bias2[1]));
          product(nt + step, q4_pair<1>(a, s2[0], bias2[0]), q4_pair<1>(c, s2[1], bias2[1]));
          product(nt + 2 * step, q4_pair<2>(a, s2[0], bias2[0]), q4_pair<2>(c, s2[1], bias2[1]));
          product(nt + 3 * step, q4_pair<3>(a, s2[0], bias2[0]), q4_pair<3>(c, s2[1], bias2[1]));
        }
      }
    }
  }
  // ---- merge the warps
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) s_acc[warp][g][q4_dim_of<NG>(nt, 2 * t + e)] = acc[nt][e] + acc[nt][e + 2];
  if (t == 0) {
    s_ml[warp][g][0] = m * prm.scale_log2;
    s_ml[warp][g][1] = l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < gc * 32 * NG; i += 32 * DQ_WARPS) {
    const int h = i / (32 * NG), d = i % (32 * NG);
    float mx = s_ml[0][h][0];
#pragma unroll
    for (int w = 1; w < DQ_WARPS; ++w) mx = fmaxf(mx, s_ml[w][h][0]);
    const float m_ref = mx == -INFINITY ? 0.f : mx;
    float a = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < DQ_WARPS; ++w) {
      const float f = ptx::ex2(s_ml[w][h][0] - m_ref);
      a = fmaf(f, s_acc[w][h][d], a);
      sum = fmaf(f, s_ml[w][h][1], sum);
    }
    if (prm.n_splits == 1) {
      if (d < D) rope_st(static_cast<ST*>(prm.o) + (bh0 + h) * D + d, len > 0 ? a / sum : 0.f);
      if (d == 0 && prm.lse != nullptr) prm.lse[bh0 + h] = len > 0 ? (mx + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    } else {
      const size_t ps = (bh0 + h) * prm.n_splits + sp;
      if (d < D) prm.part_o[ps * D + d] = a;
      if (d == 0) {
        prm.part_ml[ps * 2] = mx;
        prm.part_ml[ps * 2 + 1] = sum;
      }
    }
  }
}

// One CTA per (batch, head) adds up the splits' parts.  A split without keys has the maximum -inf and the weight 0; a sequence
// without keys gives zeros, and -inf as its log-sum-exp.
template <typename ST>
__global__ void __launch_bounds__(128)
fa_decode_q4_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const int* __restrict__ lengths, ST* __restrict__ o,
                          float* __restrict__ lse, int n_splits, int H, int D) {
  const size_t bh = blockIdx.x;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const bool empty = lengths[bh / H] <= 0;
  const float2* ml = reinterpret_cast<const float2*>(part_ml) + bh * n_splits;
  float mx = -INFINITY;
  for (int s = 0; s < n_splits; ++s) mx = fmaxf(mx, ml[s].x);
  const float m_ref = mx == -INFINITY ? 0.f : mx;
  float a = 0.f, sum = 0.f;
  const int d = threadIdx.x;
  for (int s = 0; s < n_splits; ++s) {
    const float f = ptx::ex2(ml[s].x - m_ref);
    sum = fmaf(f, ml[s].y, sum);
    if (d < D) a = fmaf(f, part_o[(bh * n_splits + s) * D + d], a);
  }
  if (d < D) rope_st(o + bh * D + d, empty ? 0.f : a / sum);
  if (d == 0 && lse != nullptr) lse[bh] = empty ? -INFINITY : (mx + log2f(sum)) * 0.6931471805599453f;
}

}  // namespace it
