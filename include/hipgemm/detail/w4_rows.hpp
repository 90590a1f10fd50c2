// Products of 5 rows of 16-bit activations and more with 4-bit weights, while
// the weights' bytes are what they cost: Stream over all of K.
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

// Items: m tiles of up to rows_max rows, parts of K (len), 32 columns of y.  With
// more than one part the sums go to o (parts x M x N) and k_w4_sum ends the work.
struct W4RowsArgs {
  W4Args a;
  float* o;
  int rows_max, parts, len;
};

template <int kX, int kW, int kS>
__device__ __forceinline__ void finish_w4(const W4Args& g, int m, int n, float f) {
  if (!(__builtin_fabsf(f) < __builtin_inff())) f = slow_row<kX, kW, kS>(g, m, n);
  if (g.bias) f += g.bias[n];
  store_result(g.y, m * g.ldy + n, g.out, activate(f, g.act));
}

template <int kX, int kW, int kS, int kMode, int kMT>
__global__ __launch_bounds__(512) void k_w4_rows(W4RowsArgs r) {
  using S = Stream<kX, kW, kS, kMode, kMT, false>;
  __shared__ __attribute__((aligned(16))) uint8_t lds[S::kXBytes];
  __shared__ __attribute__((aligned(1024))) uint8_t rings[S::kRingBytes];
  __shared__ float sums[S::kSums];
  struct Policy {
    S st;
    const W4RowsArgs& r;
    int tiles;
    __device__ __forceinline__ int group(int item) const { return item / tiles; }
    __device__ __forceinline__ int k_begin(int item) const {
      return item / tiles % r.parts * r.len;
    }
    __device__ __forceinline__ int m_begin(int q) const { return q / r.parts * r.rows_max; }
    __device__ __forceinline__ int rows(int q) const {
      return min(r.a.M - m_begin(q), r.rows_max);
    }
    __device__ __forceinline__ const uint8_t* row_at(int q, int, int m) const {
      return r.a.x + (long long)(m_begin(q) + m) * r.a.ldx;
    }
    __device__ __forceinline__ void weights(int item) {
      const int n0 = item % tiles * S::kTile;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        // (a second tile that is not there: the first one again, not used)
        const int first = min(n0 + 16 * n, (r.a.N - 1) & ~15);
        st.set_tile(n, r.a.w + (long long)first * r.a.ldw, r.a.N - first);
        const long long row = min(n0 + 16 * st.scale_tile(n) + (lane_id() & 15), r.a.N - 1);
        st.sp[n] = r.a.s + row * r.a.lds;
        if constexpr (kW == kWInt4Z) st.zp[n] = r.a.z + row * r.a.ldz;
      }
    }
    __device__ __forceinline__ void finish(int item) {
      const int q = item / tiles, n0 = (item - q * tiles) * S::kTile, n_rows = rows(q);
      for (int i = (int)threadIdx.x; i < n_rows * S::kTile; i += S::kThreads) {
        const int c = i % S::kTile, row = i / S::kTile, n = n0 + c, m = m_begin(q) + row;
        if (n >= r.a.N) continue;
        const float f = st.sum_of(c / 16, row / 16, row % 16, c % 16);
        if (r.parts > 1) r.o[((long long)(q % r.parts) * r.a.M + m) * r.a.N + n] = f;
        else finish_w4<kX, kW, kS>(r.a, m, n, f);
      }
    }
  };
  Policy p{{}, r, (r.a.N + S::kTile - 1) / S::kTile};
  p.st.lds = (lds_u8*)lds;
  p.st.rings = (lds_u8*)rings;
  p.st.sums = (__attribute__((address_space(3))) float*)sums;
  p.st.K = r.a.K;
  p.st.ldw = (uint32_t)r.a.ldw;
  p.st.inv = 32.0f / (float)r.a.G;
  const int items = (r.a.M + r.rows_max - 1) / r.rows_max * r.parts * p.tiles;
  p.st.run((int)((long long)items * blockIdx.x / gridDim.x),
           (int)((long long)items * (blockIdx.x + 1) / gridDim.x), r.len, p);
}

template <int kX, int kW, int kS>
__global__ __launch_bounds__(256) void k_w4_sum(W4RowsArgs r) {
  const int n = (int)blockIdx.x * 256 + (int)threadIdx.x, m = (int)blockIdx.y;
  if (n >= r.a.N) return;
  float f = 0.0f;
  for (int q = 0; q < r.parts; ++q) f += r.o[((long long)q * r.a.M + m) * r.a.N + n];
  finish_w4<kX, kW, kS>(r.a, m, n, f);
}

}  // namespace detail
}  // namespace hipgemm
