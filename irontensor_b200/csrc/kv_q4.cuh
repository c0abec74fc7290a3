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

// round(x / s), ties to even, in the low byte of each c, for s of at most 8 significant bits and quotients of less than 127.5; inv =
// 1 / s.  The whole number q comes out of the low bits of a sum with 1.5 * 2^23, rounded once.  x * inv may be off by a last
// place, which matters next to the middle of two whole numbers: there x - q s, exact (at most 24 bits above the last place of x),
// says which is nearer.  That is rare, and asked once for all N.
template <int N>
__device__ __forceinline__ void quant_codes(const float (&x)[N], float s, float inv, uint32_t (&c)[N]) {
  constexpr float MAGIC = 12582912.f;
  const float half = 0.5f * s;
  bool close = false;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float y = fmaf(x[e], inv, MAGIC);
    c[e] = __float_as_uint(y);
    close |= fabsf(fmaf(-(y - MAGIC), s, x[e])) >= half;
  }
  if (close) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float r = fmaf(-(__uint_as_float(c[e]) - MAGIC), s, x[e]);
      if (fabsf(r) > half || (fabsf(r) == half && (c[e] & 1u))) c[e] += r > 0.f ? 1u : 0xFFFFFFFFu;
    }
  }
}

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
// (x & MASK) | magic in one instruction.  It takes one constant in itself and no second one, so `magic` comes in a register; left to
// itself the compiler makes two instructions of it, and attention waits for the unit that executes them.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t q4_and_or(uint32_t x, uint32_t magic) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(x), "n"(MASK), "r"(magic));
  return d;
}
__device__ __forceinline__ uint32_t q4_constant(uint32_t c) {   // one that the compiler does not see through
  uint32_t d;
  asm volatile("mov.b32 %0, %1;" : "=r"(d) : "r"(c));
  return d;
}
// Nibble I of both halves of w as the values (16 + u) s - 24 s.
template <int I>
__device__ __forceinline__ uint32_t q4_pair(uint32_t w, uint32_t s2, uint32_t bias2, uint32_t magic) {
  const uint32_t at3 = I == 0 ? w << 3 : w >> (4 * I - 3);
  return q4_fma2(q4_and_or<0x00780078u>(at3, magic), s2, bias2);
}
constexpr uint32_t Q4_MAGIC = 0x41804180u;       // 16 in both halves
constexpr uint32_t Q4_MINUS_24 = 0xC1C0C1C0u;

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

// What 8 columns of a thread become: the word of their codes, and the group's scale.  The threads of a quad hold a group.
__device__ __forceinline__ uint32_t q4_quantise(const float (&x)[8], float* scale) {
  uint32_t largest = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) largest = max(largest, __float_as_uint(x[e]) & 0x7FFFFFFFu);
  largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
  largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
  float s = quant_scale<7, 5>(largest);
  const bool saturates = s > Q4_MOST_SCALE;
  if (saturates) s = Q4_MOST_SCALE;
  *scale = s;
  if (!(s > 0.f)) return 0x88888888u;   // zeros, or not numbers
  const float inv = __frcp_rn(s);
  float y[8];
  uint32_t c[8], word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = saturates ? fminf(fmaxf(x[e], -7.f * s), 7.f * s) : x[e];
  quant_codes(y, s, inv, c);
#pragma unroll
  for (int e = 0; e < 8; ++e) word |= ((c[e] + 8u) & 15u) << (4 * (e >> 1) + 16 * (e & 1));
  return word;
}

// New tokens k, v [batch, T, kv_heads, head_dim] into the cache behind the lengths[b] positions that are there; of sequence b the
// first counts[b] tokens (null: all T).  new_lengths[b] = what is there afterwards.  Grid (rows, batch, keys or values); a
// thread takes 8 columns.  Positions outside the cache are not written, and reported.
// Reads 2 * 8 or 4 * 8 bytes a thread and writes 4.5: bound by memory, and for single tokens by the launch.
template <typename ST, int NG>
__global__ void __launch_bounds__(256)
kv_q4_append_kernel(const ST* __restrict__ k, const ST* __restrict__ v, KvQ4 ck, KvQ4 cv, const int* __restrict__ lengths,
                    const int* __restrict__ counts, int* __restrict__ new_lengths, int B, int T, int Hkv, int D, int max_len, int* status) {
  constexpr int LANES = 4 * NG, ROWS = 256 / LANES;   // threads of a row, rows of a CTA
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int in_cta = static_cast<int>(threadIdx.x) / LANES, lane = static_cast<int>(threadIdx.x) % LANES, j = lane >> 2, t = lane & 3;
  const uint32_t row = blockIdx.x * ROWS + in_cta;    // of the sequence: token and head
  const int tok = static_cast<int>(row / static_cast<uint32_t>(Hkv)), h = static_cast<int>(row - static_cast<uint32_t>(tok) * Hkv);
  const int d0 = 32 * j + 8 * t;
  const ST* src = blockIdx.z ? v : k;
  const KvQ4& c = blockIdx.z ? cv : ck;
  for (int b = blockIdx.y; b < B; b += static_cast<int>(gridDim.y)) {
    const int have = lengths[b], want = counts != nullptr ? counts[b] : T, add = min(max(want, 0), T);
    if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
      const long long end = static_cast<long long>(have) + add;
      if (have < 0 || end > max_len || add != want) atomicCAS(status, 0, DEV_ERR_CACHE_RANGE);
      new_lengths[b] = static_cast<int>(min(max(end, 0LL), static_cast<long long>(max_len)));
    }
    const long long pos = static_cast<long long>(have) + tok;
    const bool live = in_cta < ROWS && tok < add && pos >= 0 && pos < max_len;
    if (!__any_sync(0xffffffffu, live)) continue;
    float x[8] = {};
    if (live && d0 < D) q4_load8(src + ((static_cast<size_t>(b) * T + tok) * Hkv + h) * D + d0, x);
    float s;
    const uint32_t word = q4_quantise(x, &s);
    if (live) {
      const size_t crow = (static_cast<size_t>(b) * Hkv + h) * max_len + pos;
      c.codes[crow * LANES + t * NG + j] = word;
      if (t == 0) c.scales[crow * NG + j] = __float2bfloat16_rn(s);
    }
  }
}

// Positions starts[b] + t, t < T, of the cache (null: from 0) as keys and values [batch, T, kv_heads, head_dim]; zeros outside
// 0 <= position < min(lengths[b], max_len) (null: max_len).  Grid as above; a thread writes 8 columns.  Bound by the bytes that it
// writes.
template <typename ST, int NG>
__global__ void __launch_bounds__(256)
kv_q4_read_kernel(ST* __restrict__ k, ST* __restrict__ v, KvQ4 ck, KvQ4 cv, const int* __restrict__ starts, const int* __restrict__ lengths,
                  int B, int T, int Hkv, int D, int max_len) {
  constexpr int LANES = 4 * NG, ROWS = 256 / LANES;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int in_cta = static_cast<int>(threadIdx.x) / LANES, lane = static_cast<int>(threadIdx.x) % LANES, j = lane >> 2, t = lane & 3;
  const uint32_t row = blockIdx.x * ROWS + in_cta;
  const int tok = static_cast<int>(row / static_cast<uint32_t>(Hkv)), h = static_cast<int>(row - static_cast<uint32_t>(tok) * Hkv);
  const int d0 = 32 * j + 8 * t;
  if (in_cta >= ROWS || tok >= T || d0 >= D) return;
  ST* dst = blockIdx.z ? v : k;
  const KvQ4& c = blockIdx.z ? cv : ck;
  for (int b = blockIdx.y; b < B; b += static_cast<int>(gridDim.y)) {
    const long long pos = static_cast<long long>(starts != nullptr ? starts[b] : 0) + tok;
    const int end = lengths != nullptr ? min(lengths[b], max_len) : max_len;
    uint32_t x[4] = {0u, 0u, 0u, 0u};   // pairs of neighbouring columns
    if (pos >= 0 && pos < end) {
      const size_t crow = (static_cast<size_t>(b) * Hkv + h) * max_len + pos;
      const uint32_t w = __ldg(c.codes + crow * LANES + t * NG + j);
      const uint32_t s2 = __byte_perm(*reinterpret_cast<const unsigned short*>(c.scales + crow * NG + j), 0, 0x1010), bias2 = q4_mul2(s2, Q4_MINUS_24);
      x[0] = q4_pair<0>(w, s2, bias2, Q4_MAGIC);
      x[1] = q4_pair<1>(w, s2, bias2, Q4_MAGIC);
      x[2] = q4_pair<2>(w, s2, bias2, Q4_MAGIC);
      x[3] = q4_pair<3>(w, s2, bias2, Q4_MAGIC);
    }
    ST* at = dst + ((static_cast<size_t>(b) * T + tok) * Hkv + h) * D + d0;
    if constexpr (sizeof(ST) == 2) {
      *reinterpret_cast<uint4*>(at) = make_uint4(x[0], x[1], x[2], x[3]);
    } else {
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(x[i] << 16);
        f[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
      }
      q4_store8(at, f);
    }
  }
}

}  // namespace it
