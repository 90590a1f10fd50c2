// Products of 5 rows of 16-bit activations and more with 4-bit weights, while
// the weights' bytes are what they cost: Stream over all of K, K dealt to the
// waves of a workgroup and summed in LDS.
#pragma once

#include "w4_stream.hpp"
#include "w4_vec.hpp"

namespace hipgemm {
namespace detail {

// One output by its definition, weight by weight, where the sum came out
// infinite or NaN: int4's excess (decode.hpp) makes inf - inf of an infinite x,
// and the sums before the scale can overflow for one near the largest, where the
// definition has an infinity or a number.
template <int kX, int kW, int kS>
__device__ __forceinline__ float slow_row(const W4Args& g, int m, int n) {
  float sum = 0.0f;
#pragma unroll 1
  for (int k = 0; k < g.K; k += 2) {
    const int grp = k / g.G;
    const uint32_t c = g.w[n * g.ldw + (k >> 1)];
    const f32x2 x = unpack2<kX>(reinterpret_cast<const uint32_t*>(g.x + m * g.ldx)[k >> 1]);
    const float s = scale_at<kS>(g.s + n * g.lds, grp);
    const float z = g.z ? (float)g.z[n * g.ldz + grp] : 8.0f;
    sum = __builtin_fmaf(x[0], s * code_value<kW>(c & 15u, z), sum);
    sum = __builtin_fmaf(x[1], s * code_value<kW>(c >> 4, z), sum);
  }
  return sum;
}

template <int kX, int kW, int kS, int kMode, int kNT, int kMT>
__global__ __launch_bounds__(512, 2) void k_w4_rows(W4Args g) {
  const int wave = wave_id(), lane = lane_id(), waves = (int)(blockDim.x / kWave);
  const int n0 = (int)blockIdx.x * 16 * kNT, m0 = (int)blockIdx.y * 16 * kMT;
  Stream<kX, kW, kS, kMode, kNT, kMT, false> st;
  st.K = g.K;
  st.lo = 0;
  st.inv = 32.0f / (float)g.G;
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    const long long r = min(n0 + 16 * n + (lane & 15), g.N - 1);
    st.w[n] = g.w + r * g.ldw;
    st.s[n] = g.s + r * g.lds;
    st.z[n] = g.z ? g.z + r * g.ldz : nullptr;
  }
#pragma unroll
  for (int m = 0; m < kMT; ++m)
    st.x[m] = g.x + (long long)min(m0 + 16 * m + (lane & 15), g.M - 1) * g.ldx;
  st.run(wave, st.pairs(), waves);

  // Lane l, element e of tile (n, m): row 16 m + 4 (l / 16) + e, column 16 n + l % 16.
  __shared__ f32x4 part[8 * kNT * kMT * kWave];
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int m = 0; m < kMT; ++m) part[(wave * kNT * kMT + n * kMT + m) * kWave + lane] = st.acc[n][m];
  __syncthreads();
  for (int t = wave; t < kNT * kMT; t += waves) {
    f32x4 v = part[t * kWave + lane];
    for (int w = 1; w < waves; ++w) v += part[(w * kNT * kMT + t) * kWave + lane];
    const int n = n0 + 16 * (t / kMT) + (lane & 15);
    const int m = m0 + 16 * (t % kMT) + 4 * (lane >> 4);
    if (n >= g.N) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (m + e >= g.M) break;
      float f = v[e];
      if (!(__builtin_fabsf(f) < __builtin_inff()))
        f = slow_row<kX, kW, kS>(g, m + e, n);
      if (g.bias) f += g.bias[n];
      store_result(g.y, (m + e) * g.ldy + n, g.out, activate(f, g.act));
    }
  }
}

}  // namespace detail
}  // namespace hipgemm
