// The experts of a few tokens that share few of them, in two kernels of w4_vec.hpp's kind:
//
//   k_moe_vec_up    h[p] = weights[p] act(x W13[e][:F]^T) (x W13[e][F:]^T)
//   k_moe_vec_down  y[t] = sum_j h[t k + j] W2[e]^T
//
// Each pair of a token and an expert is a product of a matrix with a vector, so
// there is nothing to group: blockIdx.y names the pair (or, going down, the
// token).  Going down a workgroup takes its rows of W2 for all of the token's
// experts, dealt to its waves by expert and chunk of F, so that the sum over the
// experts is the sum over the waves in LDS, in a fixed order.  h is kH bf16 parts
// (moe.hpp), here rows of x whose sums are added.
#pragma once

#include "moe.hpp"

namespace hipgemm {
namespace detail {

template <int kX, int kW, int kS, int kLk>
__global__ __launch_bounds__(512) void k_moe_vec_up(MoeArgs g) {
  using V = Vec<kX, kW, kS, 1, kLk>;
  const int wave = wave_id(), tid = (int)threadIdx.x, p = (int)blockIdx.y;
  const int e = g.ids[p];
  if (e < 0 || e >= g.E) return;
  // Waves: along K, then gate or up, then rows of their own.
  const int wk = wave % g.waves_k, half = wave / g.waves_k % 2, wr = wave / g.waves_k / 2;
  const int f0 = (int)blockIdx.x * g.rows;
  const int r0 = f0 + wr * g.wave_rows, r1 = min(min(r0 + g.wave_rows, f0 + g.rows), g.F);
  __shared__ float part[8][kVecMaxRows];
  for (int i = tid; i < 8 * kVecMaxRows; i += (int)blockDim.x) (&part[0][0])[i] = 0.0f;
  __syncthreads();
  const uint8_t* x = g.x + (long long)(p / g.k) * g.ldx;
  const long long up = half ? g.F : 0;
  V v;
  for (int k0 = wk * V::kChunk; k0 < g.D; k0 += g.waves_k * V::kChunk)
    if (r0 < r1)
      v.pass(k0, g.D, g.G, [&](int) { return x; }, g.w13 + e * g.w13_expert + up * g.w13_row,
             g.w13_row, g.s13 + e * g.s13_expert + up * g.s13_row, g.s13_row,
             kW == kWInt4Z ? g.z13 + e * g.z13_expert + up * g.z13_row : nullptr, g.z13_row, r0,
             r1, part[wave]);
  __syncthreads();
  for (int i = tid; i < g.rows; i += (int)blockDim.x) {
    const int f = f0 + i, q = i / g.wave_rows, at = i - q * g.wave_rows;
    if (f >= g.F) continue;
    float a = 0.0f, b = 0.0f;
    for (int w = 0; w < g.waves_k; ++w) {
      a += part[2 * q * g.waves_k + w][at];
      b += part[(2 * q + 1) * g.waves_k + w][at];
    }
    store_h(g, p, f, activate(a, g.act) * b * g.weights[p]);
  }
}

template <int kW, int kS, int kLk, int kH>
__global__ __launch_bounds__(512) void k_moe_vec_down(MoeArgs g) {
  using V = Vec<kInBf16, kW, kS, kH, kLk>;
  const int wave = wave_id(), tid = (int)threadIdx.x, t = (int)blockIdx.y;
  const int waves = (int)blockDim.x / kWave;
  const int r0 = (int)blockIdx.x * g.rows, r1 = min(r0 + g.rows, g.D);
  __shared__ float part[8][kH * kVecMaxRows];
  for (int i = tid; i < 8 * kH * kVecMaxRows; i += (int)blockDim.x) (&part[0][0])[i] = 0.0f;
  __syncthreads();
  const int chunks = (g.F + V::kChunk - 1) / V::kChunk;
  V v;
  for (int i = wave; i < g.k * chunks; i += waves) {
    const int p = t * g.k + i / chunks;
    const int e = g.ids[p];
    if (e < 0 || e >= g.E) continue;
    const uint8_t* h = reinterpret_cast<const uint8_t*>(g.h + (long long)p * kH * g.F);
    v.pass(i % chunks * V::kChunk, g.F, g.G, [&](int m) { return h + m * 2ll * g.F; },
           g.w2 + e * g.w2_expert, g.w2_row, g.s2 + e * g.s2_expert, g.s2_row,
           kW == kWInt4Z ? g.z2 + e * g.z2_expert : nullptr, g.z2_row, r0, r1, part[wave]);
  }
  __syncthreads();
  for (int i = tid; i < r1 - r0; i += (int)blockDim.x) {
    float f = 0.0f;
    for (int w = 0; w < waves; ++w)
#pragma unroll
      for (int q = 0; q < kH; ++q) f += part[w][q * kVecMaxRows + i];
    store_result(g.y, t * g.ldy + r0 + i, g.out, f);
  }
}

}  // namespace detail
}  // namespace hipgemm
