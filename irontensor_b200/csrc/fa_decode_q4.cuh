// Attention for one new token per sequence against a 4-bit key/value cache (kv_q4.cuh), every sequence at its own length:
// o[b, h] = softmax(q[b, h] K^T / sqrt(D)) V over the first lengths[b] positions of K/V head h / (heads / kv_heads).
//
// A value of the cache is c * s, exact in bf16.  A nibble u = c + 8 masked into the upper mantissa bits of a bf16 whose exponent
// says 16 is the number 16 + u, and (16 + u) * s - 24 * s = c * s is one fma of two packed values, exact because 24 * s has 7
// significant bits and c * s at most 8.  So a 32-bit word of eight codes becomes four operand registers by a shift, a mask and an
// fma each, and everything behind that is bf16 matrix instructions (mma.sync m16n8k16, fp32 sums):
//   S^T = K Q^T   A: 16 keys by 16 columns, which lie together in a word of the cache; B: the columns of 8 query heads
//   O^T = V^T P^T A: 16 columns by 16 keys.  A register holds one column of two keys, so two keys' words are interleaved by
//                 halves first (four byte permutes for 32 codes); B: P of 16 keys and 8 heads, S^T transposed in 8 x 8 tiles
// with the codes as the larger operand, so that an instruction's 16 rows are all in use whatever the number of heads.
// P goes in as two bf16 terms, 16 bits, which is 2^-17 of each p: of the bf16 results for B32 H32/8 D128 ragged to 8190, 0.2 % are not
// the nearest to the exact value, where sums in plain fp32 leave 0.07 %, and both are 0.00166 away from it (the rounding to bf16 itself).
// A third term would be half of V's matrix instructions again, and with PAIRED columns as many.  An fp32 q goes in as three terms, as does its P.  Where a K/V head has up
// to four query heads and q is bf16, these are there twice among the instruction's eight columns, and P's terms are its columns 0-3
// and 4-7: half the instructions for O (PAIRED; the same case: 51 -> 48.5 us when it came).
// Which key is which row of S^T, and which column of V is which row of O^T, is free as long as both products agree: the order
// is the one in which the words lie (q4_dim_of, q4_key_of).
//
// What has to be read is 144 bytes a position of a K/V head at head_dim 128: 23 us of the 47.7 that the case above takes, 3.2 TB/s
// (sixteen sequences of 16000: 74.7 us, 3.9 TB/s).  No unit is full: over 32 sequences of 8192 the schedulers issue in 61 % of the
// cycles, the integer unit is busy in 53 %, the matrix unit in 22 %, with 706 instructions for the 32 keys that a warp takes at a time.
// A block of keys is one chain (codes, scores, vote, exponentials, transposes, values), a scheduler has fewer than three warps, and in
// 40 % of the cycles none of them can go on; registers leave no room for a fourth.  tcgen05 makes the chain longer: the operands are
// made all the same, and go through shared or tensor memory and a wait for each tile: 75 us where this took 46.5.  So
//   * a warp has a ring of three stages of 32 keys in shared memory, filled by asynchronous copies that nobody but it waits for;
//     no barrier until a CTA's warps merge what they found;
//   * long caches: a persistent launch (PLAN_EVEN), in which every CTA takes the same number of 32-key units of the whole batch,
//     whatever the sequences' lengths, which only the device knows: it adds them up and finds its own stretch.  A stretch that
//     ends inside a sequence leaves its part for fa_decode_q4_merge_kernel.  A CTA has at most two such parts, so the
//     workspace does not grow with the batch;
//   * short ones (PLAN_CLUSTER): even shares of a sequence on the 1 to 8 CTAs of a cluster, merged through distributed shared
//     memory in the same launch, which saves the second one.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "gemm_skinny.cuh"
#include "kv_q4.cuh"
#include "sm100_ptx.cuh"

namespace it {

constexpr int DQ_BLOCK = 32, DQ_STAGES = 3, DQ_MAX_CTAS = 512, DQ_START = 12;
enum : int { PLAN_CLUSTER = 0, PLAN_EVEN = 1 };
// Warps of a CTA and CTAs of an SM.  The persistent launches of bf16 have three CTAs of four warps: up to 168 registers a thread, which the loop
// needs more than it needs a fourth warp on each scheduler with 128 and some of them in memory (B32 H32/8 D128 ragged to 8190, where this
// was 46.5 us: with eight warps twice 2.5 more, six warps twice 2), and few warps that wait for one another where a stretch ends.
__host__ __device__ constexpr bool dq_threes(int terms, int heads, int plan) { return plan == PLAN_EVEN && terms == 1 && heads == 8; }
__host__ __device__ constexpr int dq_warps(int terms, int heads, int plan) { return dq_threes(terms, heads, plan) ? 4 : 8; }
__host__ __device__ constexpr int dq_ctas(int terms, int heads, int plan) { return dq_threes(terms, heads, plan) ? 3 : terms == 1 && heads == 8 ? 2 : 1; }
constexpr int DQ_MERGE_WARPS = 8;

struct DecodeQ4Params {
  const void* q;            // [batch, heads, D]
  const uint32_t *k_codes, *v_codes;
  const __nv_bfloat16 *k_scales, *v_scales;
  const int* lengths;
  void* o;
  float *lse, *part_o, *part_ml;
  int* units;               // PLAN_EVEN: work in front of each sequence [batch + 1], and a CTA's share, for the merge
  int* status;
  int B, H, Hkv, D, max_len;
  int n_splits;             // PLAN_CLUSTER: CTAs of a cluster
  float scale_log2;         // 1/sqrt(D) * log2(e)
};

// D = A B + C in fp16 with fp32 sums.
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                              float c0, float c1, float c2, float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t q4_add2_f16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Which column of a head is row r (0 .. 15) of O^T's m-tile mt (see the V operand below).
template <int NG>
__device__ __forceinline__ int q4_dim_of(int mt, int r) {
  constexpr int F = NG / 2;
  const int n = r & 7;
  int w, i;
  if (mt < 4 * F) {
    w = n * F + mt / 4;                  // whole sets of 8 words: lane n owns F consecutive words
    i = mt % 4;
  } else {
    w = 8 * F + (n & 3);                 // the last 4 words, of which lanes 4-7 take the upper columns
    i = mt - 4 * F + 2 * (n >> 2);
  }
  return 32 * (w % NG) + 8 * (w / NG) + 2 * i + (r >> 3);
}

__device__ __forceinline__ uint32_t transposed_8x8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}

template <int NG>
struct DecodeQ4Stage {
  static constexpr int CODES = DQ_BLOCK * 16 * NG;                          // of 32 rows
  static constexpr int SCALES = (DQ_BLOCK * 2 * NG + 2 + 15) / 16 * 16;     // and up to two bytes in front of them
  static constexpr int BYTES = 2 * CODES + 2 * SCALES;
  static constexpr int WARP_BYTES = DQ_STAGES * BYTES;
};

// Position in the block of a score's column: the n-th of 8 is key n / 2 (n even) or 4 + (n / 2 ^ X).  With the V operand's
// rows (the keys of columns 2t and 2t + 1) as they then come, loads of both operands are free of bank conflicts.
template <int NG>
__device__ __forceinline__ int q4_key_of(int n) {
  return (n & 1) ? 4 + ((n >> 1) ^ (NG == 2 ? 2 : 1)) : n >> 1;
}
// Rows of 64 bytes: 16-byte chunk c of row r lies at chunk c ^ 2 ((r / 2) % 2), see q4_key_of.
template <int NG>
__device__ __forceinline__ int q4_chunk(int r, int c) { return NG == 4 ? c ^ ((r & 2)) : c; }

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, int bytes) {   // of N bytes; zeros behind `bytes`
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Copies the codes and scales of `n` rows (of which 32 at most) from `first` on of one half of a cache into a stage.  Chunk
// 32 u + lane of the codes is row 8 u + lane / 4 where rows have four, whose place in the swizzle is the lane's alone.
template <int NG>
__device__ __forceinline__ void q4_fetch(uint32_t codes_at, uint32_t scales_at, const uint32_t* codes, const __nv_bfloat16* scales, size_t first,
                                         int n, int lane) {
  const char* src = reinterpret_cast<const char*>(codes) + first * (16 * NG) + lane * 16;
  const uint32_t dst = codes_at + (NG == 4 ? (lane >> 2) * 4 + q4_chunk<4>(lane >> 2, lane & 3) : lane) * 16;
  if (n >= DQ_BLOCK) {
#pragma unroll
    for (int u = 0; u < NG; ++u) cp_async_16(dst + u * 512, src + u * 512);
  } else {
#pragma unroll
    for (int u = 0; u < NG; ++u)
      if (u * 32 + lane < n * NG) cp_async_16(dst + u * 512, src + u * 512);
  }
  const char* sc = reinterpret_cast<const char*>(scales) + first * (2 * NG);
  if constexpr (NG % 2 == 0) {
    if (lane < n) cp_async_small<2 * NG>(scales_at + lane * 2 * NG, sc + lane * 2 * NG, 2 * NG);
  } else {   // rows of 2 or 6 bytes: whole words from the boundary in front of the first
    const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(sc) & 2), bytes = min(n, DQ_BLOCK) * 2 * NG + lead;
    for (int at = lane * 4; at < bytes; at += 128) cp_async_small<4>(scales_at + at, sc - lead + at, min(4, bytes - at));
  }
}

// The running softmax and output of one warp, of 8 R query heads; PAIRED: of four, columns h and h + 4 being the upper and the lower
// term of head h.
template <int NG, int TERMS, int R, bool PAIRED>
struct DecodeQ4Warp {
  static_assert(!PAIRED || (TERMS == 1 && R == 1), "two terms of P, eight columns");
  static constexpr int PT = PAIRED ? 1 : TERMS == 1 ? 2 : 3;   // instructions for P's terms
  static constexpr int MT = 2 * NG;
  float acc[MT][R][4];   // of m-tile, 8 heads: rows g and g + 8 by heads 2t and 2t + 1
  // Of heads 2t and 2t + 1: what p is relative to, the score above which that is renewed, and this lane's keys' share of the sum.
  // p is exp2(score - m) with an m that may lie up to RANGE below the largest score: sums and products keep their relative
  // precision, and after the first keys a renewal is rare.
  static constexpr float RANGE = 8.f;   // in the exp2 domain
  float m[R][2], limit[R][2], l[R][2];
  // fp32 q: K's values are made in bf16 like V's, and q has three bf16 terms.  bf16 q: K's codes alone are the operand, in fp16,
  // whose ten bits of mantissa take two nibbles by a mask each, the known way of making numbers of them: u in the lowest is 1024 + u and u in the next is 64 + u, less 1032 and
  // 72 by an addition, both exact.  A shift by 8 brings the other two.  (Adding 72 times the sum of q to the sums instead would save
  // half of the additions, and leave in a score 2^-24 of that, whatever small codes the score is made of.)
  // So a word costs five instructions of the integer unit and not eight; its scale is applied to the sums of its 32 columns in fp32.  q is scaled by a power of two to a largest magnitude in 1 .. 2 for this (fp16 rounds what is below 2^-14
  // of the largest, by at most 2^-25 of it).
  static constexpr bool F16 = TERMS == 1;
  uint32_t magic, magic0, magic1;
  uint32_t qb[TERMS][R][4 * NG];    // register 4 j + r: columns 32 j + 8 t + 2 r and the next of head g
  float scale[R][2];                // of the scores of these heads, in the exp2 domain

  __device__ __forceinline__ void begin() {
    magic = q4_constant(Q4_MAGIC);
    magic0 = q4_constant(0x64006400u);   // 1024 in fp16
    magic1 = q4_constant(0x54005400u);   // 64
#pragma unroll
    for (int h = 0; h < R; ++h) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][h][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[h][e] = limit[h][e] = -INFINITY;
        l[h][e] = 0.f;
      }
    }
  }
  // q: the first of the heads; scale_log2 = 1/sqrt(D) * log2(e)
  template <typename ST>
  __device__ __forceinline__ void load_q(const ST* q, int heads, int D, float scale_log2, int g, int t) {
#pragma unroll
    for (int h = 0; h < R; ++h) {
      const int head = PAIRED ? g & 3 : 8 * h + g;
      const bool live = head < heads;
      const ST* row = q + head * D;
      if constexpr (F16) {
        uint32_t largest = 0;
#pragma unroll
        for (int i = 0; i < 4 * NG; ++i) {
          const int d = 32 * (i >> 2) + 8 * t + 2 * (i & 3);
          qb[0][h][i] = live && d < D ? *reinterpret_cast<const uint32_t*>(row + d) : 0u;
          largest = max(largest, max(qb[0][h][i] & 0x7FFFu, (qb[0][h][i] >> 16) & 0x7FFFu));
        }
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // 2^-e for the exponent e of the largest; 1 for zeros and where something is not finite
        const uint32_t field = largest >> 7;
        const bool as_is = field == 0 || field == 255;
        const float down = as_is ? 1.f : __uint_as_float((254u - min(field, 253u)) << 23), up = as_is ? 1.f : __uint_as_float(min(field, 253u) << 23);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            uint32_t& x = qb[0][h][4 * j + r];
            const __half2 y = __floats2half2_rn(__uint_as_float(x << 16) * down, __uint_as_float(x & 0xFFFF0000u) * down);
            x = *reinterpret_cast<const uint32_t*>(&y);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) scale[h][e] = scale_log2 * __shfl_sync(0xffffffffu, up, 8 * t + 4 * e);
      } else {
#pragma unroll
        for (int i = 0; i < 4 * NG; ++i) {
          const int d = 32 * (i >> 2) + 8 * t + 2 * (i & 3);
          float x0 = 0.f, x1 = 0.f;
          if (live && d < D) {
            x0 = rope_ld(row + d);
            x1 = rope_ld(row + d + 1);
          }
#pragma unroll
          for (int n = 0; n < TERMS; ++n) {
            qb[n][h][i] = ptx::pack_bf16(x0, x1);
            x0 -= __uint_as_float(qb[n][h][i] << 16);
            x1 -= __uint_as_float(qb[n][h][i] & 0xFFFF0000u);
          }
        }
        scale[h][0] = scale[h][1] = scale_log2;
      }
    }
  }

  // `n` keys (at most 32) of the stage at `stage`; k_lead, v_lead: where a row's scales begin, in elements behind the stage's.
  __device__ __forceinline__ void block(const uint8_t* stage, int n, int k_lead, int v_lead, int g, int t) {
    using S = DecodeQ4Stage<NG>;
    const unsigned short* ks = reinterpret_cast<const unsigned short*>(stage + 2 * S::CODES) + k_lead;
    const unsigned short* vs = reinterpret_cast<const unsigned short*>(stage + 2 * S::CODES + S::SCALES) + v_lead;
    const int key = q4_key_of<NG>(g);   // in 8; 8 more rows do not change a row's swizzle
    const uint32_t* k_row = reinterpret_cast<const uint32_t*>(stage) + key * 4 * NG + (NG == 4 ? 4 * q4_chunk<NG>(key, t) : t * NG);
    const unsigned short* k_scale = ks + key * NG;
    float s[2][R][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {   // 16 keys: rows g and g + 8
      uint32_t w[2][NG], sc[2][NG];   // a scale in the low half of its register
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int first = 16 * i + 8 * x;
        const uint32_t* src = k_row + first * 4 * NG;
        if constexpr (NG == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(src);
          w[x][0] = v.x, w[x][1] = v.y, w[x][2] = v.z, w[x][3] = v.w;
          const uint2 u = *reinterpret_cast<const uint2*>(k_scale + first * 4);
          sc[x][0] = u.x, sc[x][1] = u.x >> 16, sc[x][2] = u.y, sc[x][3] = u.y >> 16;
        } else if constexpr (NG == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(src);
          w[x][0] = v.x, w[x][1] = v.y;
          const uint32_t u = *reinterpret_cast<const uint32_t*>(k_scale + first * 2);
          sc[x][0] = u, sc[x][1] = u >> 16;
        } else {
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            w[x][j] = src[j];
            sc[x][j] = k_scale[first * NG + j];
          }
        }
      }
#pragma unroll
      for (int h = 0; h < R; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][h][e] = 0.f;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        if constexpr (F16) {
          constexpr uint32_t LESS = 0xE408E408u, LESS1 = 0xD480D480u;   // -1032 and -72 in fp16
          const uint32_t u0 = w[0][j] >> 8, u1 = w[1][j] >> 8;
          const uint32_t a0 = q4_add2_f16(q4_and_or<0x000F000Fu>(w[0][j], magic0), LESS), a1 = q4_add2_f16(q4_and_or<0x000F000Fu>(w[1][j], magic0), LESS);
          const uint32_t a2 = q4_add2_f16(q4_and_or<0x00F000F0u>(w[0][j], magic1), LESS1), a3 = q4_add2_f16(q4_and_or<0x00F000F0u>(w[1][j], magic1), LESS1);
          const uint32_t a4 = q4_add2_f16(q4_and_or<0x000F000Fu>(u0, magic0), LESS), a5 = q4_add2_f16(q4_and_or<0x000F000Fu>(u1, magic0), LESS);
          const uint32_t a6 = q4_add2_f16(q4_and_or<0x00F000F0u>(u0, magic1), LESS1), a7 = q4_add2_f16(q4_and_or<0x00F000F0u>(u1, magic1), LESS1);
          const float f0 = __uint_as_float(sc[0][j] << 16), f1 = __uint_as_float(sc[1][j] << 16);
#pragma unroll
          for (int h = 0; h < R; ++h) {
            float d[4];
            mma_f16_16816(d, a0, a1, a2, a3, qb[0][h][4 * j], qb[0][h][4 * j + 1], 0.f, 0.f, 0.f, 0.f);
            mma_f16_16816(d, a4, a5, a6, a7, qb[0][h][4 * j + 2], qb[0][h][4 * j + 3], d[0], d[1], d[2], d[3]);
            s[i][h][0] = fmaf(f0, d[0], s[i][h][0]);
            s[i][h][1] = fmaf(f0, d[1], s[i][h][1]);
            s[i][h][2] = fmaf(f1, d[2], s[i][h][2]);
            s[i][h][3] = fmaf(f1, d[3], s[i][h][3]);
          }
        } else {
          const uint32_t s0 = __byte_perm(sc[0][j], 0, 0x1010), s1 = __byte_perm(sc[1][j], 0, 0x1010);
          const uint32_t bias0 = q4_mul2(s0, Q4_MINUS_24), bias1 = q4_mul2(s1, Q4_MINUS_24);
          const uint32_t a0 = q4_pair<0>(w[0][j], s0, bias0, magic), a1 = q4_pair<0>(w[1][j], s1, bias1, magic);
          const uint32_t a2 = q4_pair<1>(w[0][j], s0, bias0, magic), a3 = q4_pair<1>(w[1][j], s1, bias1, magic);
          const uint32_t a4 = q4_pair<2>(w[0][j], s0, bias0, magic), a5 = q4_pair<2>(w[1][j], s1, bias1, magic);
          const uint32_t a6 = q4_pair<3>(w[0][j], s0, bias0, magic), a7 = q4_pair<3>(w[1][j], s1, bias1, magic);
#pragma unroll
          for (int h = 0; h < R; ++h)
#pragma unroll
            for (int x = TERMS - 1; x >= 0; --x) {
              mma_bf16_16816(s[i][h], a0, a1, a2, a3, qb[x][h][4 * j], qb[x][h][4 * j + 1]);
              mma_bf16_16816(s[i][h], a4, a5, a6, a7, qb[x][h][4 * j + 2], qb[x][h][4 * j + 3]);
            }
        }
      }
    }
    if (n < DQ_BLOCK) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (16 * i + 8 * (e >> 1) + key >= n)
#pragma unroll
            for (int h = 0; h < R; ++h) s[i][h][e] = -INFINITY;
    }
    // online softmax; a lane holds 4 of the 32 keys of each of its two heads
    uint32_t p[PT][R][4];   // terms of P, transposed: register x of keys 8x .. 8x + 7
#pragma unroll
    for (int h = 0; h < R; ++h) {
      float mx[2], m_ref[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) mx[e] = fmaxf(ptx::fmax3(s[0][h][e], s[0][h][e + 2], s[1][h][e]), s[1][h][e + 2]);
      if (__any_sync(0xffffffffu, mx[0] > limit[h][0] || mx[1] > limit[h][1])) {
        float corr[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(mx[e], m[h][e]);
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 4));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 8));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 16));
          corr[e] = mx[e] > m[h][e] ? ptx::ex2((m[h][e] - mx[e]) * scale[h][e]) : 1.f;
          l[h][e] *= corr[e];
          m[h][e] = mx[e];
          limit[h][e] = mx[e] + RANGE / scale[h][e];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][h][e] *= corr[e & 1];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) m_ref[e] = m[h][e] == -INFINITY ? 0.f : m[h][e] * scale[h][e];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float p0 = ptx::ex2(fmaf(s[x >> 1][h][2 * (x & 1)], scale[h][0], -m_ref[0]));
        float p1 = ptx::ex2(fmaf(s[x >> 1][h][2 * (x & 1) + 1], scale[h][1], -m_ref[1]));
        l[h][0] += p0;
        l[h][1] += p1;
        if constexpr (PAIRED) {
          const uint32_t upper = ptx::pack_bf16(p0, p1);
          const uint32_t lower = ptx::pack_bf16(p0 - __uint_as_float(upper << 16), p1 - __uint_as_float(upper & 0xFFFF0000u));
          p[0][h][x] = transposed_8x8(t < 2 ? upper : lower);
        } else {
#pragma unroll
          for (int y = 0; y < PT; ++y) {
            const uint32_t term = ptx::pack_bf16(p0, p1);
            p0 -= __uint_as_float(term << 16);
            p1 -= __uint_as_float(term & 0xFFFF0000u);
            p[y][h][x] = transposed_8x8(term);
          }
        }
      }
    }
    // O^T += V^T P^T, 16 keys at a time
    constexpr int F = NG / 2, HALF = NG & 1;   // whole sets of 8 words; a set of 4
    const uint32_t* v_row[2];
    const unsigned short* v_scale[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {   // keys 2t and 2t + 1
      const int row = q4_key_of<NG>(2 * t + x);
      v_row[x] = reinterpret_cast<const uint32_t*>(stage + S::CODES) + row * 4 * NG + (NG == 4 ? 4 * q4_chunk<NG>(row, g >> 1) + 2 * (g & 1) : 0);
      v_scale[x] = vs + row * NG + (NG == 4 ? 2 * (g & 1) : 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t w[4][F + HALF], sc[4][F + HALF];   // by key (2t, 2t + 1, 2t + 8, 2t + 9) and set of words; scales in the low half
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int first = 16 * i + 8 * (x >> 1);
        const uint32_t* src = v_row[x & 1] + first * 4 * NG;
        const unsigned short* scales = v_scale[x & 1] + first * NG;
        if constexpr (NG == 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(src);
          w[x][0] = v.x, w[x][1] = v.y;
          const uint32_t u = *reinterpret_cast<const uint32_t*>(scales);
          sc[x][0] = u, sc[x][1] = u >> 16;
        } else {
#pragma unroll
          for (int f = 0; f < F + HALF; ++f) {
            const int word = f < F ? g * F + f : 8 * F + (g & 3);
            w[x][f] = src[word];
            if (f >= F) w[x][f] >>= 8 * (g >> 2);   // lanes 4-7: the upper two nibbles of each half
            sc[x][f] = scales[word % NG];
          }
        }
      }
#pragma unroll
      for (int f = 0; f < F + HALF; ++f) {
        uint32_t s2[2], bias2[2], lo[2], hi[2];   // the low halves of two keys' words are even columns, the high halves odd ones
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          s2[x] = __byte_perm(sc[2 * x][f], sc[2 * x + 1][f], 0x5410);
          bias2[x] = q4_mul2(s2[x], Q4_MINUS_24);
          lo[x] = __byte_perm(w[2 * x][f], w[2 * x + 1][f], 0x5410);
          hi[x] = __byte_perm(w[2 * x][f], w[2 * x + 1][f], 0x7632);
        }
        auto product = [&](int mt, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
          for (int h = 0; h < R; ++h)
#pragma unroll
            for (int y = PT - 1; y >= 0; --y) mma_bf16_16816(acc[mt][h], a0, a1, a2, a3, p[y][h][2 * i], p[y][h][2 * i + 1]);
        };
        product(4 * f, q4_pair<0>(lo[0], s2[0], bias2[0], magic), q4_pair<0>(hi[0], s2[0], bias2[0], magic), q4_pair<0>(lo[1], s2[1], bias2[1], magic),
                q4_pair<0>(hi[1], s2[1], bias2[1], magic));
        product(4 * f + 1, q4_pair<1>(lo[0], s2[0], bias2[0], magic), q4_pair<1>(hi[0], s2[0], bias2[0], magic), q4_pair<1>(lo[1], s2[1], bias2[1], magic),
                q4_pair<1>(hi[1], s2[1], bias2[1], magic));
        if (f < F) {
          product(4 * f + 2, q4_pair<2>(lo[0], s2[0], bias2[0], magic), q4_pair<2>(hi[0], s2[0], bias2[0], magic), q4_pair<2>(lo[1], s2[1], bias2[1], magic),
                  q4_pair<2>(hi[1], s2[1], bias2[1], magic));
          product(4 * f + 3, q4_pair<3>(lo[0], s2[0], bias2[0], magic), q4_pair<3>(hi[0], s2[0], bias2[0], magic), q4_pair<3>(lo[1], s2[1], bias2[1], magic),
                  q4_pair<3>(hi[1], s2[1], bias2[1], magic));
        }
      }
    }
  }

  // What the warp found: its output relative to its maximum, by head and row of O^T, that maximum in the exp2 domain, and the sum.
  // With PITCH rows a head the 32 lanes' stores lie in different banks.
  static constexpr int PITCH = 32 * NG + 4;
  __device__ __forceinline__ void leave(float* out /* [8 R][PITCH] */, float (*ml)[2], int g, int t) {
#pragma unroll
    for (int h = 0; h < R; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[h][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int head = 8 * h + 2 * t + e;
        if (g == 0) {
          ml[head][0] = m[h][e] * scale[h][e];
          ml[head][1] = sum;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float upper = acc[mt][h][e], lower = acc[mt][h][e + 2];   // rows g and g + 8
          if constexpr (PAIRED) {
            upper += __shfl_xor_sync(0xffffffffu, upper, 2);
            lower += __shfl_xor_sync(0xffffffffu, lower, 2);
            if (t >= 2) continue;
          }
          out[head * PITCH + 16 * mt + g] = upper;
          out[head * PITCH + 16 * mt + g + 8] = lower;
        }
      }
  }
};

// NG: groups of 32 columns; TERMS: bf16 terms of q (1: bf16 q, two-term P; 3: fp32 q, three-term P); HEADS: query heads of a CTA, 8
// or, in bf16, 16, which share the operands made of the codes; PAIRED: there are four at most.
// PLAN_CLUSTER: grid (n_splits, kv_heads * chunks, batch), clusters of n_splits.  PLAN_EVEN: any number of CTAs up to DQ_MAX_CTAS.
template <int NG, int TERMS, int HEADS, bool PAIRED, int PLAN>
__global__ void __launch_bounds__(32 * dq_warps(TERMS, HEADS, PLAN), dq_ctas(TERMS, HEADS, PLAN))
fa_decode_q4_kernel(const DecodeQ4Params prm) {
  using ST = typename std::conditional<TERMS == 1, __nv_bfloat16, float>::type;
  using S = DecodeQ4Stage<NG>;
  using Warp = DecodeQ4Warp<NG, TERMS, HEADS / 8, PAIRED>;
  constexpr int DQ_WARPS = dq_warps(TERMS, HEADS, PLAN), COLS = 32 * NG, STEP = DQ_WARPS * DQ_BLOCK;
  // A warp leaves its output in the one stage of its ring that is free, while the first keys of the CTA's next stretch are on
  // their way into the others; 16 heads take the whole ring.
  constexpr bool AHEAD = HEADS == 8 && PLAN == PLAN_EVEN;
  static_assert(HEADS * Warp::PITCH * 4 <= (AHEAD ? S::BYTES : S::WARP_BYTES) && S::BYTES % 16 == 0, "room for a warp's output");
  extern __shared__ __align__(16) uint8_t dq_smem[];
  __shared__ float s_ml[DQ_WARPS][HEADS][2], s_weight[DQ_WARPS][HEADS], s_total[HEADS][2];
  __shared__ uint32_t s_left[DQ_WARPS];    // where the warps' outputs are
  __shared__ int s_scan[DQ_WARPS + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = prm.H / prm.Hkv, chunks = (G + HEADS - 1) / HEADS, per_b = prm.Hkv * chunks, D = prm.D;
  uint8_t* ring = dq_smem + warp * S::WARP_BYTES;
  const uint32_t ring_at = ptx::smem_addr(ring);
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();

  auto length_of = [&](int b) {
    const int given = prm.lengths[b], len = min(max(given, 0), prm.max_len);
    if (given != len) atomicCAS(prm.status, 0, DEV_ERR_CACHE_RANGE);
    return len;
  };
  // Keys k0 .. k1 - 1 of sequence b and pair p (of K/V head and head chunk).
  struct Stretch {
    int b, p, k0, k1;
  };
  auto row_of = [&](const Stretch& x) { return (static_cast<size_t>(x.b) * prm.Hkv + x.p / chunks) * prm.max_len; };
  auto heads_of = [&](const Stretch& x) { return min(HEADS, G - (x.p % chunks) * HEADS); };
  auto bh_of = [&](const Stretch& x) { return static_cast<size_t>(x.b) * prm.H + (x.p / chunks) * G + (x.p % chunks) * HEADS; };
  Warp w;
  // The warp's blocks on their way: of the stretch at hand, or of the one behind it.
  int fetch_k = 0, fetch_end = 0, on_way = 0;
  size_t fetch_row = 0;
  uint32_t put = 0, take = 0;
  auto next_stage = [](uint32_t at) { return at == (DQ_STAGES - 1) * S::BYTES ? 0u : at + S::BYTES; };
  auto fetch_from = [&](const Stretch& x) {
    fetch_k = x.k0 + warp * DQ_BLOCK;
    fetch_end = x.k1;
    fetch_row = row_of(x);
  };
  auto fetch = [&] {
    if (!AHEAD && fetch_k >= fetch_end) cp_async_commit();   // an empty group, so that the groups count the steps
    if (fetch_k >= fetch_end || (AHEAD && on_way == DQ_STAGES)) return;
    const uint32_t at = ring_at + put;
    const int n = fetch_end - fetch_k;
    q4_fetch<NG>(at, at + 2 * S::CODES, prm.k_codes, prm.k_scales, fetch_row + fetch_k, n, lane);
    q4_fetch<NG>(at + S::CODES, at + 2 * S::CODES + S::SCALES, prm.v_codes, prm.v_scales, fetch_row + fetch_k, n, lane);
    cp_async_commit();
    fetch_k += STEP;
    put = next_stage(put);
    if (AHEAD) ++on_way;
  };
  // Attends to a stretch by all warps and leaves their results in the rings; `next` is what comes behind it (k1 = 0: nothing).
  // Called with the first blocks on their way, and fetch_k within the stretch.
  auto attend = [&](const Stretch& x, const Stretch& next) {
    const size_t row0 = row_of(x);
    bool behind = false;    // fetch_k is in the next stretch
    auto fetch_on = [&] {
      if (AHEAD && !behind && fetch_k >= fetch_end) {
        fetch_from(next);
        behind = true;
      }
      fetch();
    };
    auto lead = [&](const __nv_bfloat16* scales, int k0) {
      return NG % 2 == 0 ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(scales + (row0 + k0) * NG) & 2) / 2;
    };
    w.load_q(static_cast<const ST*>(prm.q) + bh_of(x) * D, heads_of(x), D, prm.scale_log2, g, t);
    w.begin();
    for (int k0 = x.k0 + warp * DQ_BLOCK; k0 < x.k1; k0 += STEP) {
      if (AHEAD && on_way < 2) fetch_on();
      if (!AHEAD || on_way > 1) cp_async_wait<1>();
      else cp_async_wait<0>();
      __syncwarp();    // the block is there for all lanes, and all have done with the one before it
      fetch_on();
      uint8_t* stage = ring + take;
      const int n = x.k1 - k0, kl = lead(prm.k_scales, k0), vl = lead(prm.v_scales, k0);
      if (n < DQ_BLOCK) {   // the rows behind the last key keep what was there: scales of zero make them nothing
        if (lane >= n) {
          unsigned short* ks = reinterpret_cast<unsigned short*>(stage + 2 * S::CODES) + kl + lane * NG;
          unsigned short* vs = reinterpret_cast<unsigned short*>(stage + 2 * S::CODES + S::SCALES) + vl + lane * NG;
#pragma unroll
          for (int j = 0; j < NG; ++j) ks[j] = vs[j] = 0;
        }
        __syncwarp();
      }
      w.block(stage, n, kl, vl, g, t);
      take = next_stage(take);
      if (AHEAD) --on_way;
    }
    if (!AHEAD) {
      cp_async_wait<0>();
      put = take = 0;
    }
    __syncwarp();
    if (!behind && AHEAD) fetch_from(next);
    const uint32_t left = AHEAD ? put : 0u;     // on_way < DQ_STAGES here: the stage at `put` is free
    if (lane == 0) s_left[warp] = warp * S::WARP_BYTES + left;
    w.leave(reinterpret_cast<float*>(ring + left), s_ml[warp], g, t);
    __syncthreads();
    // the warps' results as one: weights, then four rows a thread
    if (threadIdx.x < DQ_WARPS * HEADS) {
      const int y = threadIdx.x / HEADS, h = threadIdx.x % HEADS;
      float mx = s_ml[0][h][0], sum = 0.f;
#pragma unroll
      for (int z = 1; z < DQ_WARPS; ++z) mx = fmaxf(mx, s_ml[z][h][0]);
      const float m_ref = mx == -INFINITY ? 0.f : mx;
      s_weight[y][h] = ptx::ex2(s_ml[y][h][0] - m_ref);
      if (y == 0) {
#pragma unroll
        for (int z = 0; z < DQ_WARPS; ++z) sum = fmaf(ptx::ex2(s_ml[z][h][0] - m_ref), s_ml[z][h][1], sum);
        s_total[h][0] = mx;
        s_total[h][1] = sum;
      }
    }
    __syncthreads();
  };
  // f(head, first of four rows of O^T, their outputs) for all of the CTA's result; s_total has the maxima and sums.
  auto merged = [&](int heads, auto&& f) {
    for (int i = threadIdx.x; i < heads * (COLS / 4); i += 32 * DQ_WARPS) {
      const int h = i / (COLS / 4), r = 4 * (i % (COLS / 4));
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < DQ_WARPS; ++x) {
        const float e = s_weight[x][h];
        const float4 v = *reinterpret_cast<const float4*>(dq_smem + s_left[x] + (h * Warp::PITCH + r) * 4);
        a.x = fmaf(e, v.x, a.x);
        a.y = fmaf(e, v.y, a.y);
        a.z = fmaf(e, v.z, a.z);
        a.w = fmaf(e, v.w, a.w);
      }
      f(h, r, a);
    }
  };
  auto store_o = [&](size_t bh, int r, float x) {
    const int d = q4_dim_of<NG>(r >> 4, r & 15);
    if (d < D) rope_st(static_cast<ST*>(prm.o) + bh * D + d, x);
  };
  auto store_lse = [&](size_t bh, float mx, float sum, bool some) {
    if (prm.lse != nullptr) prm.lse[bh] = some ? (mx + log2f(sum)) * 0.6931471805599453f : -INFINITY;
  };
  auto finish = [&](size_t bh0, int heads, bool some) {
    merged(heads, [&](int h, int r, const float4& a) {
      const float sum = s_total[h][1], inv = some ? 1.f / sum : 0.f;
      store_o(bh0 + h, r, a.x * inv);
      store_o(bh0 + h, r + 1, a.y * inv);
      store_o(bh0 + h, r + 2, a.z * inv);
      store_o(bh0 + h, r + 3, a.w * inv);
      if (r == 0) store_lse(bh0 + h, s_total[h][0], sum, some);
    });
  };

  if constexpr (PLAN == PLAN_CLUSTER) {
    const int b = blockIdx.z, p = blockIdx.y, sp = blockIdx.x, n = prm.n_splits;
    const int len = length_of(b), blocks = (len + DQ_BLOCK - 1) / DQ_BLOCK, share = (blocks + n - 1) / n;
    const Stretch x{b, p, min(sp * share * DQ_BLOCK, len), min((sp + 1) * share * DQ_BLOCK, len)};
    const int heads = heads_of(x);
    const size_t bh0 = bh_of(x);
    fetch_from(x);
    fetch();
    fetch();
    attend(x, Stretch{0, 0, 0, 0});
    if (n == 1) {
      finish(bh0, heads, len > 0);
      return;
    }
    // The CTA's result takes the place of its first warp's: four rows are read, and then written, by one thread alone.
    float* c_acc = reinterpret_cast<float*>(dq_smem);
    merged(heads, [&](int h, int r, const float4& a) { *reinterpret_cast<float4*>(c_acc + h * Warp::PITCH + r) = a; });
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int i = sp + static_cast<int>(threadIdx.x) * n; i < heads * COLS; i += 32 * DQ_WARPS * n) {
      const int h = i / COLS, r0 = i - h * COLS;
      float ms[8], ls[8], as[8], mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        ms[r] = -INFINITY;
        if (r < n) {
          const float* ml = cluster.map_shared_rank(&s_total[h][0], r);
          ms[r] = ml[0];
          ls[r] = ml[1];
          as[r] = *cluster.map_shared_rank(c_acc + h * Warp::PITCH + r0, r);
        }
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) mx = fmaxf(mx, ms[r]);
      const float m_ref = mx == -INFINITY ? 0.f : mx;
      float a = 0.f, sum = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < n) {
          const float e = ptx::ex2(ms[r] - m_ref);
          a = fmaf(e, as[r], a);
          sum = fmaf(e, ls[r], sum);
        }
      store_o(bh0 + h, r0, len > 0 ? a / sum : 0.f);
      if (r0 == 0) store_lse(bh0 + h, mx, sum, len > 0);
    }
    cluster.sync();   // nobody's shared memory goes away while it is read
  } else {
    // The work of a pair is its units of 32 keys and DQ_START units for beginning and ending it: without those, a CTA whose
    // share is many short sequences would be the last by far (32 sequences of up to 2000 positions: 59 us, with them 24).
    // All CTAs add up the work in front of each sequence, and find the one that their own share begins in.
    constexpr int threads = 32 * DQ_WARPS;
    auto work_of = [&](int len) { return len > 0 ? DQ_START + (len + DQ_BLOCK - 1) / DQ_BLOCK : 0; };   // of one pair
    int total = 0, share = 0, first = 0;
    const int chunks_b = (prm.B + threads - 1) / threads;
    for (int pass = chunks_b > 1 ? 0 : 1; pass < 2; ++pass) {   // a batch of more than one chunk is gone through twice
      int before = 0;
      for (int c = 0; c < chunks_b; ++c) {
        const int b = c * threads + static_cast<int>(threadIdx.x);
        const int work = b < prm.B ? per_b * work_of(length_of(b)) : 0;
        int incl = work;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, incl, off);
          if (lane >= off) incl += up;
        }
        if (lane == 31) s_scan[warp] = incl;
        __syncthreads();
        int at = before + incl - work;
#pragma unroll
        for (int x = 0; x < DQ_WARPS; ++x) {
          if (x < warp) at += s_scan[x];
          before += s_scan[x];
        }
        if (pass == 1) {
          if (chunks_b == 1) total = before;
          share = max((total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), DQ_START + DQ_WARPS);
          first = min(static_cast<int>(blockIdx.x) * share, total);
          if (b < prm.B) {
            if (first >= at && first < at + work) {
              s_scan[DQ_WARPS] = b;
              s_scan[DQ_WARPS + 1] = at;
            }
            if (blockIdx.x == 0) prm.units[b] = at;
          }
        }
        __syncthreads();
      }
      total = before;
    }
    const int last = min(first + share, total);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      prm.units[prm.B] = total;
      prm.units[prm.B + 1] = share;
    }
    if (first >= last) return;
    int b = s_scan[DQ_WARPS], at = s_scan[DQ_WARPS + 1], u = first;
    // The share's next stretch (k1 = 0: none), and whether it is a whole sequence.
    auto next_stretch = [&](bool* whole) {
      while (u < last) {
        const int len = min(max(prm.lengths[b], 0), prm.max_len), per_pair = work_of(len);
        if (u >= at + per_b * per_pair) {
          at += per_b * per_pair;
          ++b;
          continue;
        }
        const int p = (u - at) / per_pair, begin = at + p * per_pair + DQ_START, end = begin + per_pair - DQ_START;
        const int u0 = max(u, begin), u1 = min(last, end);   // of the pair's units of keys begin .. end - 1
        u = end;
        if (u0 >= u1) continue;
        *whole = u0 == begin && u1 == end;
        return Stretch{b, p, (u0 - begin) * DQ_BLOCK, min((u1 - begin) * DQ_BLOCK, len)};
      }
      return Stretch{0, 0, 0, 0};
    };
    bool whole = false, next_whole = false;
    Stretch x = next_stretch(&whole);
    fetch_from(x);
    fetch();
    fetch();
    while (x.k1 > 0) {
      const Stretch next = next_stretch(&next_whole);
      attend(x, next);
      const int heads = heads_of(x);
      if (whole) {
        finish(bh_of(x), heads, true);
      } else {
        const size_t part = (2 * static_cast<size_t>(blockIdx.x) + (x.k0 == 0 ? 1 : 0)) * HEADS;   // begun here, or in front of it
        merged(heads, [&](int h, int r, const float4& a) {
          *reinterpret_cast<float4*>(prm.part_o + (part + h) * COLS + r) = a;
          if (r == 0) {
            prm.part_ml[(part + h) * 2] = s_total[h][0];
            prm.part_ml[(part + h) * 2 + 1] = s_total[h][1];
          }
        });
      }
      __syncthreads();   // the rings are filled again
      if (!AHEAD) fetch_from(next);
      if (!AHEAD || on_way < 2) fetch();
      if (!AHEAD || on_way < 2) fetch();
      x = next;
      whole = next_whole;
    }
  }
}

// PLAN_EVEN: adds up the parts of a sequence that more than one CTA worked on.  Grid (batch * heads, 1 or NG): of the NG CTAs of a
// (batch, head) each takes 32 rows of O^T, where there are few (batch, head).  A warp takes every eighth part.  A sequence without
// keys gives zeros, and -inf as its log-sum-exp.
template <typename ST, int NG, int HEADS, int JN>   // JN: groups of 32 rows of a CTA, NG or 1
__global__ void __launch_bounds__(32 * DQ_MERGE_WARPS)
fa_decode_q4_merge_kernel(const DecodeQ4Params prm) {
  constexpr int COLS = 32 * NG;
  __shared__ float s_acc[DQ_MERGE_WARPS][32 * JN], s_e[DQ_MAX_CTAS], s_mx[DQ_MERGE_WARPS], s_sum[DQ_MERGE_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = static_cast<int>(blockIdx.x) / prm.H, head = static_cast<int>(blockIdx.x) % prm.H;
  const int G = prm.H / prm.Hkv, chunks = (G + HEADS - 1) / HEADS, per_b = prm.Hkv * chunks;
  const int p = head / G * chunks + head % G / HEADS, h = head % G % HEADS;
  const int j0 = static_cast<int>(blockIdx.y) * JN;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int at = prm.units[b], per_pair = (prm.units[b + 1] - at) / per_b, share = prm.units[prm.B + 1];
  const int begin = at + p * per_pair + DQ_START, c0 = begin / share, c1 = per_pair > 0 ? (at + (p + 1) * per_pair - 1) / share : c0;
  const size_t bh = blockIdx.x;
  ST* o = static_cast<ST*>(prm.o) + bh * prm.D;
  if (per_pair == 0) {
    if (blockIdx.y == 0 && threadIdx.x < prm.D) rope_st(o + threadIdx.x, 0.f);
    if (blockIdx.y == 0 && threadIdx.x == 0 && prm.lse != nullptr) prm.lse[bh] = -INFINITY;
    return;
  }
  if (c0 == c1) return;
  auto part_of = [&](int c) { return (2 * static_cast<size_t>(c) + (c == c0 ? 1 : 0)) * HEADS + h; };
  // The warp's parts are loaded some at a time, the first of them along with the maxima (one sequence of 131000 with two K/V heads, 148
  // parts a pair then: 24.6 -> 21.8 us in all; an even share of the work there is 10 us of it, the scan 0.8, a stretch's end 1.3, this
  // kernel 2.5).  28 for each of eight warps are the 222 parts that half of 444 CTAs may leave a pair.
  constexpr int AT_ONCE = JN == 1 ? 28 : 4;
  float v[AT_ONCE][JN];
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
      for (int j = 0; j < JN; ++j)
        v[i][j] = c + i * DQ_MERGE_WARPS <= c1 ? prm.part_o[part_of(c + i * DQ_MERGE_WARPS) * COLS + 32 * (j0 + j) + lane] : 0.f;
  };
  load(c0 + warp);
  float2 ml[2];   // of up to DQ_MAX_CTAS parts
  float mx = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = c0 + i * 32 * DQ_MERGE_WARPS + static_cast<int>(threadIdx.x);
    ml[i] = c <= c1 ? *reinterpret_cast<const float2*>(prm.part_ml + part_of(c) * 2) : make_float2(-INFINITY, 0.f);
    mx = fmaxf(mx, ml[i].x);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
  if (lane == 0) s_mx[warp] = mx;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < DQ_MERGE_WARPS; ++x) mx = fmaxf(mx, s_mx[x]);
  const float m_ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float e = ptx::ex2(ml[i].x - m_ref);
    s_e[i * 32 * DQ_MERGE_WARPS + threadIdx.x] = e;
    sum = fmaf(e, ml[i].y, sum);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int x = 0; x < DQ_MERGE_WARPS; ++x) sum += s_sum[x];
  float a[JN] = {};
  for (int c = c0 + warp; c <= c1; c += AT_ONCE * DQ_MERGE_WARPS) {
    if (c > c0 + warp) load(c);
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const float e = c + i * DQ_MERGE_WARPS <= c1 ? s_e[c + i * DQ_MERGE_WARPS - c0] : 0.f;
#pragma unroll
      for (int j = 0; j < JN; ++j) a[j] = fmaf(e, v[i][j], a[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < JN; ++j) s_acc[warp][32 * j + lane] = a[j];
  __syncthreads();
  const int r = 32 * j0 + static_cast<int>(threadIdx.x);
  if (threadIdx.x < 32 * JN) {
    const int d = q4_dim_of<NG>(r >> 4, r & 15);
    float total = 0.f;
#pragma unroll
    for (int x = 0; x < DQ_MERGE_WARPS; ++x) total += s_acc[x][threadIdx.x];
    if (d < prm.D) rope_st(o + d, total / sum);
  }
  if (r == 0 && prm.lse != nullptr) prm.lse[bh] = (mx + log2f(sum)) * 0.6931471805599453f;
}

}  // namespace it
