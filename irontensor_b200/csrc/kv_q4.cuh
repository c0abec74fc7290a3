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
// magnitude.  The product with 1 / MOST is right but for its last places; which side of the middle between two results the quotient
// is on is what largest and MOST * middle say, both exact.
// SHORT: `largest` of 8 significant bits.  A quotient that is no tie is then a 2^-17th and more of itself away from one, so that the
// product, right to 2^-22, is on the right side of it, and on it for ties, when it has been rounded to 19 bits.
template <int MOST, int BITS, bool SHORT>
__device__ __forceinline__ float quant_scale_inside(uint32_t largest_bits) {   // of a finite `largest` of 2^-100 and more
  constexpr int DROP = 24 - BITS;
  constexpr uint32_t MASK = (1u << DROP) - 1u, HALF = 1u << (DROP - 1);
  const float largest = __uint_as_float(largest_bits);
  if constexpr (SHORT) {
    const uint32_t q = (__float_as_uint(largest * (1.f / MOST)) + 16u) & ~31u;
    return __uint_as_float((q + (HALF - 1u) + ((q >> DROP) & 1u)) & ~MASK);
  }
  const uint32_t base = __float_as_uint(largest * (1.f / MOST)) & ~MASK;
  const float middle = static_cast<float>(MOST) * __uint_as_float(base | HALF);
  const bool up = largest > middle || (largest == middle && ((base >> DROP) & 1u));
  return __uint_as_float(base + (up ? MASK + 1u : 0u));
}
template <int MOST, int BITS>
__device__ __forceinline__ float quant_scale(uint32_t largest_bits) {
  const float s = quant_scale_inside<MOST, BITS, false>(largest_bits), largest = __uint_as_float(largest_bits);
  return largest_bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : largest < 0x1p-100f ? 0.f : s;
}

// round(x / s), ties to even, plus BIAS in the low 16 bits of each c, for s of at most 8 significant bits and quotients of less than
// 127.5; inv = 1 / s to 22 bits.  The whole number comes out of the low bits of a sum with 1.5 * 2^23, rounded once.
// SHORT: x of 8 significant bits, where ties are common.  A quotient of x and s that is no tie is 2^-11 away from one and more (they
// are whole numbers below 2^8 but for a power of two, of which quotients of a quarter and more leave few).  So x * inv, rounded to
// 14 places behind the point by a sum with 768, is on the right side of the middle between two whole numbers, and is the middle
// where x / s is: the second sum then rounds ties to even.
// Otherwise x * inv may be off by a few last places, which matters next to the middle of two whole numbers: there x - q s, exact (at
// most 24 bits above the last place of x), says which is nearer.  That is rare, and asked once for all N.
template <int BIAS, bool SHORT, int N>
__device__ __forceinline__ void quant_codes(const float (&x)[N], float s, float inv, uint32_t (&c)[N]) {
  constexpr float MAGIC = 12582912.f + BIAS;
  if constexpr (SHORT) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      c[e] = __float_as_uint(fmaf(x[e], inv, 768.f) + (MAGIC - 768.f));
    }
    return;
  }
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
      if (fabsf(r) > half || (fabsf(r) == half && ((c[e] - BIAS) & 1u))) c[e] += r > 0.f ? 1u : 0xFFFFFFFFu;
    }
  }
}
__device__ __forceinline__ float quant_inverse(float s) {
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  return inv;
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

// Eight columns as they are loaded, and the largest of their magnitudes by its bits as fp32.
template <typename ST>
struct Raw8;
template <>
struct Raw8<__nv_bfloat16> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ uint32_t largest() const {
    auto max2 = [](uint32_t a, uint32_t b) {
      uint32_t d;
      asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
      return d;
    };
    const uint32_t m = max2(max2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), max2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
    return max(m & 0xFFFF0000u, m << 16);
  }
  __device__ __forceinline__ void to(float (&x)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Raw8<float> {
  uint4 v, w;
  __device__ __forceinline__ void load(const float* p) {
    v = __ldg(reinterpret_cast<const uint4*>(p));
    w = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  }
  __device__ __forceinline__ uint32_t largest() const {
    constexpr uint32_t M = 0x7FFFFFFFu;
    return max(max(max(v.x & M, v.y & M), max(v.z & M, v.w & M)), max(max(w.x & M, w.y & M), max(w.z & M, w.w & M)));
  }
  __device__ __forceinline__ void to(float (&x)[8]) const {
    const uint32_t b[8] = {v.x, v.y, v.z, v.w, w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(b[i]);
  }
};

// What 8 columns of a thread become: the word of their codes, and the group's scale.  The threads of a quad hold a group.
template <typename ST>
__device__ __forceinline__ uint32_t q4_quantise(const Raw8<ST>& raw, float* scale) {
  uint32_t largest = raw.largest();
  largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
  largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
  float s, x[8];
  raw.to(x);
  constexpr uint32_t LEAST = 0x0D800000u, MOST = 0x7DE00000u;   // 2^-100; 7 * Q4_MOST_SCALE
  if (largest - LEAST <= MOST - LEAST) {
    s = quant_scale_inside<7, 5, sizeof(ST) == 2>(largest);
  } else if (largest < LEAST || largest >= 0x7F800000u) {       // zeros, or not numbers
    *scale = largest < LEAST ? 0.f : __uint_as_float(0x7FC00000u);
    return 0x88888888u;
  } else {
    s = Q4_MOST_SCALE;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fminf(fmaxf(x[e], -7.f * s), 7.f * s);
  }
  *scale = s;
  uint32_t c[8], p[4];
  quant_codes<8, sizeof(ST) == 2>(x, s, quant_inverse(s), c);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __byte_perm(c[2 * i], c[2 * i + 1], 0x5410);
  return (p[0] + 16u * p[1]) + 256u * (p[2] + 16u * p[3]);
}

constexpr int KV_ROWS_A_THREAD = 4;   // whose loads are in flight together

// Where a thread of the two kernels below is: 8 columns of tokens `tok`, `tok` + at_once, ... of one head.  A CTA takes at_once tokens
// of ROWS / at_once heads at a time: all of its rows are one head's where there are that many tokens.  (Walking the heads of a token
// instead reads the source in one piece and divides at every row: 10 % slower.)
template <int NG>
struct KvLane {
  static constexpr int LANES = 4 * NG, ROWS = 256 / LANES;   // threads of a row, rows of a CTA at a time
  int j, t, tok, head;
  bool in;
  __device__ __forceinline__ explicit KvLane(int at_once) {
    const int row = static_cast<int>(threadIdx.x) / LANES;
    j = static_cast<int>(threadIdx.x) % LANES >> 2;
    t = static_cast<int>(threadIdx.x) & 3;
    head = row / at_once;
    in = head < ROWS / at_once;
    tok = static_cast<int>(blockIdx.x) * (at_once * KV_ROWS_A_THREAD) + row - head * at_once;
  }
};

// New tokens k, v [batch, T, kv_heads, head_dim] into the cache behind the lengths[b] positions that are there; of sequence b the
// first counts[b] tokens (null: all T).  new_lengths[b] = what is there afterwards.  Grid (tokens, batch * kv_heads, keys or values).
// Positions outside the cache are not written, and reported.
// Bound by memory, 2 or 4 bytes read and 0.56 written a value, with the instructions close behind (8 x 2999 tokens of 8 heads of 128 in bf16:
// 23.8 us, 5.3 TB/s; with twice the instructions a value 37), and for single tokens by the launch.
// FULL: at_once is ROWS, known to the compiler.
template <typename ST, int NG, bool FULL>
__global__ void __launch_bounds__(256)
kv_q4_append_kernel(const ST* __restrict__ k, const ST* __restrict__ v, KvQ4 ck, KvQ4 cv, const int* __restrict__ lengths,
                    const int* __restrict__ counts, int* __restrict__ new_lengths, int B, int T, int Hkv, int D, int max_len, int at_once, int* status) {
  using L = KvLane<NG>;
  constexpr int U = KV_ROWS_A_THREAD;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  if (FULL) at_once = L::ROWS;
  const L at(at_once);
  const int heads = L::ROWS / at_once;   // of a CTA
  const int d0 = 32 * at.j + 8 * at.t;
  const ST* src = blockIdx.z ? v : k;
  const KvQ4& c = blockIdx.z ? cv : ck;
  for (int bh0 = static_cast<int>(blockIdx.y) * heads; bh0 < B * Hkv; bh0 += static_cast<int>(gridDim.y) * heads) {
    const bool in = at.in && bh0 + at.head < B * Hkv;
    const int bh = in ? bh0 + at.head : bh0, b = bh / Hkv, h = bh - b * Hkv;
    const int have = lengths[b], want = counts != nullptr ? counts[b] : T, add = min(max(want, 0), T);
    if (blockIdx.z == 0 && in && h == 0 && at.tok == 0 && at.j == 0 && at.t == 0) {
      const long long end = static_cast<long long>(have) + add;
      if (have < 0 || end > max_len || add != want) atomicCAS(status, 0, DEV_ERR_CACHE_RANGE);
      new_lengths[b] = static_cast<int>(min(max(end, 0LL), static_cast<long long>(max_len)));
    }
    // tokens lo .. lo + span - 1 go to positions of the cache
    const int lo = have < 0 ? -max(have, -INT32_MAX) : 0;
    const int hi = static_cast<int>(max(min(static_cast<long long>(add), static_cast<long long>(max_len) - have), 0LL));
    const unsigned span = in && hi > lo ? hi - lo : 0;
    const int stride = static_cast<int>(gridDim.x) * U * at_once;
    const size_t row0 = static_cast<size_t>(static_cast<long long>(bh) * max_len + have + at.tok), step = static_cast<size_t>(at_once) * Hkv * D;
    const ST* from = src + ((static_cast<size_t>(b) * T + at.tok) * Hkv + h) * D + d0;
    uint32_t* codes = c.codes + row0 * L::LANES + at.t * NG + at.j;
    __nv_bfloat16* scales = c.scales + row0 * NG + at.j;
    for (int tok = at.tok;;) {
      Raw8<ST> x[U] = {};
      bool live[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        live[u] = static_cast<unsigned>(tok + u * at_once - lo) < span;
        if (live[u] && d0 < D) x[u].load(from + u * step);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!__any_sync(0xffffffffu, live[u])) continue;
        float s;
        const uint32_t word = q4_quantise(x[u], &s);
        if (live[u]) {
          codes[u * at_once * L::LANES] = word;
          if (at.t == 0) scales[u * at_once * NG] = __float2bfloat16_rn(s);
        }
      }
      if (__all_sync(0xffffffffu, tok >= hi - stride)) break;
      tok += stride;
      from += static_cast<size_t>(stride) * Hkv * D;
      codes += static_cast<size_t>(stride) * L::LANES;
      scales += static_cast<size_t>(stride) * NG;
    }
  }
}

// Positions starts[b] + t, t < T, of the cache (null: from 0) as keys and values [batch, T, kv_heads, head_dim]; zeros outside
// 0 <= position < min(lengths[b], max_len) (null: max_len).  Grid as above.  Bound by the bytes that it writes.
template <typename ST, int NG>
__global__ void __launch_bounds__(256)
kv_q4_read_kernel(ST* __restrict__ k, ST* __restrict__ v, KvQ4 ck, KvQ4 cv, const int* __restrict__ starts, const int* __restrict__ lengths,
                  int B, int T, int Hkv, int D, int max_len, int at_once) {
  using L = KvLane<NG>;
  constexpr int U = KV_ROWS_A_THREAD;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const L at(at_once);
  const int heads = L::ROWS / at_once;   // of a CTA
  const int d0 = 32 * at.j + 8 * at.t;
  ST* dst = blockIdx.z ? v : k;
  const KvQ4& c = blockIdx.z ? cv : ck;
  for (int bh0 = static_cast<int>(blockIdx.y) * heads; bh0 < B * Hkv; bh0 += static_cast<int>(gridDim.y) * heads) {
    // A thread whose columns only pad a group has nothing of its own, but stays with its row: in the exchange below it stores half of
    // what its neighbour holds, at an address made from the row that both are in.
    const bool row = at.in && bh0 + at.head < B * Hkv, none = !row || d0 >= D;
    const int bh = row ? bh0 + at.head : bh0, b = bh / Hkv, h = bh - b * Hkv;
    const long long start = starts != nullptr ? starts[b] : 0;
    const int end = lengths != nullptr ? min(lengths[b], max_len) : max_len;
    uint32_t w[U], s2[U];
    const size_t crow = static_cast<size_t>(bh) * max_len + start + at.tok;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int tok = at.tok + u * at_once;
      const long long pos = start + tok;
      w[u] = 0x88888888u;
      s2[u] = 0u;
      if (!none && tok < T && pos >= 0 && pos < end) {
        const size_t r = crow + u * at_once;
        w[u] = __ldg(c.codes + r * L::LANES + at.t * NG + at.j);
        s2[u] = __ldg(reinterpret_cast<const unsigned short*>(c.scales) + r * NG + at.j);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int tok = at.tok + u * at_once;
      const bool there = !none && tok < T;
      const uint32_t s = __byte_perm(s2[u], 0, 0x1010), bias = q4_mul2(s, Q4_MINUS_24);
      const uint32_t x[4] = {q4_pair<0>(w[u], s, bias, Q4_MAGIC), q4_pair<1>(w[u], s, bias, Q4_MAGIC), q4_pair<2>(w[u], s, bias, Q4_MAGIC),
                             q4_pair<3>(w[u], s, bias, Q4_MAGIC)};   // pairs of neighbouring columns
      ST* out = dst + ((static_cast<size_t>(b) * T + tok) * Hkv + h) * D + d0;
      if constexpr (sizeof(ST) == 2) {
        if (there) *reinterpret_cast<uint4*>(out) = make_uint4(x[0], x[1], x[2], x[3]);
      } else {
        // A thread has 32 bytes and stores 16 at a time: as they lie, every store would fill half of each 32-byte sector.  So two
        // neighbours store together, first the 32 bytes of the even one and then those of the odd one.
        uint32_t f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[2 * i] = x[i] << 16;
          f[2 * i + 1] = x[i] & 0xFFFF0000u;
        }
        const bool odd = threadIdx.x & 1;
        uint32_t got[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) got[i] = __shfl_xor_sync(0xffffffffu, odd ? f[i] : f[4 + i], 1);
        const bool other = __shfl_xor_sync(0xffffffffu, static_cast<int>(there), 1) != 0;
        ST* even_at = out - (odd ? 8 : 0);   // the even thread's columns
        if (odd ? other : there) *reinterpret_cast<uint4*>(even_at + (odd ? 4 : 0)) = odd ? make_uint4(got[0], got[1], got[2], got[3]) : make_uint4(f[0], f[1], f[2], f[3]);
        if (odd ? there : other) *reinterpret_cast<uint4*>(even_at + 8 + (odd ? 4 : 0)) = odd ? make_uint4(f[4], f[5], f[6], f[7]) : make_uint4(got[0], got[1], got[2], got[3]);
      }
    }
  }
}

}  // namespace it
