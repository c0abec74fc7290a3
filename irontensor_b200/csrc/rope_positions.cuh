// Rotary embedding at positions given per token, on one or several axes (time, height and width of image and video tokens; the
// lengths of a ragged batch's sequences), and its inverse.
//
// Dimension pair i turns by   angle = positions[axis(i)][token] * f(i)   as in rope.cuh: (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos).
// The inverse turns back and is the gradient.  The pairs of a head are cut into one section per axis; f(i) and axis(i) come from
// the host.
// Angles are in 64 bits: at position 200000 an angle in 32 bits, as rope.cuh has it, is off by up to 0.01, which is 2^-7 of a
// result; here the whole turns are taken off in 64 bits and the rest of at most pi, then rounded to 32, is off by 2^-24 of itself.
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

// (cos, sin) of position * freq.  |position| < 2^31 and freq is at most a few: up to 2^30 whole turns, so the turn is given in two
// parts and the product with its first is exact in the fma.
__device__ __forceinline__ float2 rope_turn(int position, double freq) {
  const double a = static_cast<double>(position) * freq;
  const double n = rint(a * 0.15915494309189535);            // 1 / (2 pi)
  double r = fma(-n, 6.283185307179586, a);
  r = fma(-n, 2.4492935982947064e-16, r);                    // 2 pi - its first part
  float s, c;
  sincosf(static_cast<float>(r), &s, &c);
  return make_float2(c, s);
}

// A CTA owns n_pos tokens: one sine per thread into shared memory, then the heads of q and k in chunks of VEC elements (16 bytes; 2
// elements where rows are not whole chunks), of which a thread has four in flight, the first four before the sines.  A thread stays
// with one chunk of a head, `half` / (VEC / 2) threads a head, and steps over the (token, head) rows.
template <typename ST, int VEC>
__global__ void __launch_bounds__(256, 4)
rope_positions_kernel(const ST* q_in, const ST* k_in, ST* q_out, ST* k_out, const int* __restrict__ positions, long long rows, int n_pos,
                      int H, int Hkv, int D, int inverse, const __grid_constant__ RopeAxes axes) {
  constexpr int U = 4;
  __shared__ float2 tab[256];
  struct alignas(VEC * sizeof(ST)) Chunk { ST e[VEC]; };
  const int half = D >> 1, per_head = D / VEC, n_heads = H + Hkv;
  const long long row0 = static_cast<long long>(blockIdx.x) * n_pos;
  const int n_rows = static_cast<int>(min(static_cast<long long>(n_pos), rows - row0));
  const int step = 256 / per_head, mine = static_cast<int>(threadIdx.x) / per_head, d = (static_cast<int>(threadIdx.x) - mine * per_head) * VEC;
  const int step_r = step / n_heads, step_h = step - step_r * n_heads;
  int r = mine < step ? mine / n_heads : n_rows, h = mine < step ? mine - r * n_heads : 0;   // the threads behind the last whole head: none
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
        float2 cs = rope_turn(positions[axes.axis[pair] * rows + row0 + tr], axes.freq[pair]);
        if (inverse) cs.y = -cs.y;
        tab[i] = cs;
      }
      __syncthreads();
      first = false;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (rr[u] >= n_rows) break;
      const float2* cs = &tab[rr[u] * half + (d >> 1)];
#pragma unroll
      for (int p = 0; p < VEC / 2; ++p) {
        const float x0 = rope_ld(&x[u].e[2 * p]), x1 = rope_ld(&x[u].e[2 * p + 1]);
        rope_st(&x[u].e[2 * p], x0 * cs[p].x - x1 * cs[p].y);
        rope_st(&x[u].e[2 * p + 1], x0 * cs[p].y + x1 * cs[p].x);
      }
      *reinterpret_cast<Chunk*>(off[u] >= 0 ? q_out + q_at + off[u] : k_out + k_at + ~off[u]) = x[u];
    }
  }
}

}  // namespace it
