// Rotary embedding at positions given per token, on one or several axes (time, height and width of image and video tokens; the
// lengths of a ragged batch's sequences), and its inverse.
//
// Dimension pair i turns by   angle = positions[axis(i)][token] * f(i)   as in rope.cuh: (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos).
// The inverse turns back and is the gradient.  The pairs of a head are cut into one section per axis; f(i) and axis(i) come from
// the host.
// Angles are in 64 bits: at position 200000 an angle in 32 bits, as rope.cuh has it, is off by up to 0.01, which is 2^-7 of a
// result; here whole quarter turns are taken off in 64 bits and the rest, rounded to 32, is off by 2^-24 of itself.
#pragma once
#include <cuda_bf16.h>

#include <cstdint>

#include "rope.cuh"
#include "sm100_ptx.cuh"

namespace it {

struct RopeAxes {
  double freq[64];      // f(i), i < head_dim / 2
  uint8_t axis[64];
};

// A base below 1 makes frequencies above 1.  Up to this one there are at most 2^40 quarter turns to take off, and what is left is right to
// 2^-53; at 2^20 it is no longer below pi / 4, and behind 2^31 the quarters cannot be counted.
constexpr double ROPE_MOST_FREQ = 512.0;

// (cos, sin) of position * freq.  Quarter turns are taken off in 64 bits: |position| <= 2^31 and freq <= ROPE_MOST_FREQ, so there are up
// to 2^40 of them, and pi / 2 is given in two parts, the product with the first of which is exact in the fma, as is the difference.  What
// is left, at most pi / 4 and 2^-11 of it, goes through the Taylor series in 32 bits (their next terms are below 2^-29 there), and the
// quarter says which is which.
__device__ __forceinline__ float2 rope_turn(int position, double freq) {
  const double a = static_cast<double>(position) * freq;
  const double n = rint(a * 0.6366197723675814);             // 2 / pi
  double r = fma(-n, 1.5707963267948966, a);
  r = fma(-n, 6.123233995736766e-17, r);                     // pi / 2 - its first part
  const float x = static_cast<float>(r), z = x * x;
  const float s = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), x);
  const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const unsigned quarter = static_cast<unsigned>(static_cast<long long>(n)) & 3u;
  const float ca = quarter & 1u ? s : c, sa = quarter & 1u ? c : s;
  return make_float2((quarter + 1u) & 2u ? -ca : ca, quarter & 2u ? -sa : sa);
}

// A chunk of VEC elements in 32-bit words, and its pairs turned.
template <typename ST, int VEC>
struct alignas(VEC * sizeof(ST)) RopeChunk {
  static constexpr int WORDS = VEC * sizeof(ST) / 4;
  uint32_t w[WORDS];
  // c, s: the cosines and the sines of the chunk's pairs, each together and aligned to their size
  __device__ __forceinline__ void turn(const float* c, const float* s) {
    struct alignas(2 * VEC) Pairs {
      float f[VEC / 2];
    };
    const Pairs cosines = *reinterpret_cast<const Pairs*>(c), sines = *reinterpret_cast<const Pairs*>(s);
#pragma unroll
    for (int p = 0; p < VEC / 2; ++p) {
      const float2 t = make_float2(cosines.f[p], sines.f[p]);
      if constexpr (sizeof(ST) == 2) {
        const float x0 = __uint_as_float(w[p] << 16), x1 = __uint_as_float(w[p] & 0xFFFF0000u);
        w[p] = ptx::pack_bf16(x0 * t.x - x1 * t.y, x0 * t.y + x1 * t.x);
      } else {
        const float x0 = __uint_as_float(w[2 * p]), x1 = __uint_as_float(w[2 * p + 1]);
        w[2 * p] = __float_as_uint(x0 * t.x - x1 * t.y);
        w[2 * p + 1] = __float_as_uint(x0 * t.y + x1 * t.x);
      }
    }
  }
};

// A CTA owns n_pos tokens: their sines into shared memory, two per thread, then the heads of q and k in chunks of VEC elements (16 bytes; 2
// elements where rows are not whole chunks), of which a thread has four in flight, the first four before the sines.  A thread stays
// with one chunk of a head, `half` / (VEC / 2) threads a head, and steps over the (token, head) rows.
template <typename ST, int VEC>
__global__ void __launch_bounds__(256, 4)
rope_positions_kernel(const ST* q_in, const ST* k_in, ST* q_out, ST* k_out, const int* __restrict__ positions, long long rows, int n_pos,
                      int H, int Hkv, int D, int inverse, const __grid_constant__ RopeAxes axes) {
  constexpr int U = 4;
  // cosines and sines apart: a chunk's are a load of 16 bytes each, without bank conflicts (as pairs of both 17.4 -> 13.4 us for 2 x 4093
  // tokens of 16 + 4 heads of 128 in bf16 that L2 holds)
  __shared__ __align__(16) float cosines[512], sines[512];
  __shared__ double freq[64];
  __shared__ uint8_t axis[64];
  using Chunk = RopeChunk<ST, VEC>;
  const int half = D >> 1, per_head = D / VEC, n_heads = H + Hkv;
  const long long row0 = static_cast<long long>(blockIdx.x) * n_pos;
  const int n_rows = static_cast<int>(min(static_cast<long long>(n_pos), rows - row0));
  const int step = 256 / per_head, mine = static_cast<int>(threadIdx.x) / per_head, d = (static_cast<int>(threadIdx.x) - mine * per_head) * VEC;
  const int step_r = step / n_heads, step_h = step - step_r * n_heads;
  int r = mine < step ? mine / n_heads : n_rows, h = mine < step ? mine - r * n_heads : 0;   // the threads behind the last whole head: none
  // Parameters are read one address at a time: once a CTA, not once an angle (2 x 4093 tokens of 16 + 4 heads of 128 in bf16: 20.2 -> 18.5 us).
  if (threadIdx.x < half) {
    freq[threadIdx.x] = axes.freq[threadIdx.x];
    axis[threadIdx.x] = axes.axis[threadIdx.x];
  }
  __syncthreads();
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const long long q_at = row0 * H * D + d, k_at = row0 * Hkv * D + d;
  bool first = true;
  while (first || r < n_rows) {
    Chunk x[U];
    int rr[U], off[U];   // token; place in the CTA's q, or, negative, in its k
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rr[u] = r;
      off[u] = h < H ? (r * H + h) * D : ~((r * Hkv + h - H) * D);
      if (r < n_rows) x[u] = *reinterpret_cast<const Chunk*>(off[u] >= 0 ? q_in + q_at + off[u] : k_in + k_at + ~off[u]);
      r += step_r;
      h += step_h;
      if (h >= n_heads) {
        h -= n_heads;
        ++r;
      }
    }
    if (first) {   // every thread passes here once
      for (int i = static_cast<int>(threadIdx.x); i < n_rows * half; i += 256) {
        const int tr = i / half, pair = i - tr * half;
        const float2 cs = rope_turn(positions[axis[pair] * rows + row0 + tr], freq[pair]);
        cosines[i] = cs.x;
        sines[i] = inverse ? -cs.y : cs.y;
      }
      __syncthreads();
      first = false;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (rr[u] >= n_rows) break;
      x[u].turn(&cosines[rr[u] * half + (d >> 1)], &sines[rr[u] * half + (d >> 1)]);
      *reinterpret_cast<Chunk*>(off[u] >= 0 ? q_out + q_at + off[u] : k_out + k_at + ~off[u]) = x[u];
    }
  }
}

}  // namespace it
