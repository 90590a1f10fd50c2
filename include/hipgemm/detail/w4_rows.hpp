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

// A workgroup takes up to kW4Tiles tiles of 32 columns of y at a time, for a group
// of up to rows_max rows of x.  Where LDS does not hold all of K of these rows, it
// holds parts of it (len) in turn, and the tiles' sums stay in LDS from one to the
// next: x is read again for the next tiles, weights are read once.
struct W4RowsArgs {
  W4Args a;
  int rows_max, parts, len;
};
constexpr int kW4Tiles = 4;
constexpr int kW4Held = kW4Tiles * 16 * 32;  // floats per 16 rows
template <int kX, int kW, int kS, int kMode, int kMT>
using W4Stream = Stream<kX, kW, kS, kMode, kMT, false, 8, 4 * kW4Held * kMT>;

template <int kX, int kW, int kS, int kMode, int kMT>
__global__ __launch_bounds__(512) void k_w4_rows(W4RowsArgs r) {
  using S = W4Stream<kX, kW, kS, kMode, kMT>;
  __shared__ __attribute__((aligned(16))) uint8_t lds[S::kXBytes];
  __shared__ __attribute__((aligned(1024))) uint8_t rings[S::kRingBytes];
  __shared__ float sums[S::kSums];
  __shared__ float held[kW4Held * kMT];
  // Items: by batch of tiles, part of K, tile.
  struct Policy {
    S st;
    const W4RowsArgs& r;
    __attribute__((address_space(3))) float* held;
    int t0, t1;  // the workgroup's tiles, of all groups of rows
    int tiles;   // of a group
    __device__ __forceinline__ int batch(int item) const { return item / (kW4Tiles * r.parts); }
    __device__ __forceinline__ int in_batch(int b) const { return min(kW4Tiles, t1 - t0 - b * kW4Tiles); }
    __device__ __forceinline__ int part(int item) const {
      const int b = batch(item);
      return (item - b * kW4Tiles * r.parts) / in_batch(b);
    }
    __device__ __forceinline__ int slot(int item) const {
      const int b = batch(item);
      return (item - b * kW4Tiles * r.parts) % in_batch(b);
    }
    __device__ __forceinline__ int tile(int item) const {
      return t0 + batch(item) * kW4Tiles + slot(item);
    }
    __device__ __forceinline__ int k_begin(int item) const { return part(item) * r.len; }
    // Groups here: rows and part of K.
    __device__ __forceinline__ int group(int item) const {
      return tile(item) / tiles * r.parts + part(item);
    }
    __device__ __forceinline__ int m_begin(int q) const { return q / r.parts * r.rows_max; }
    __device__ __forceinline__ int rows(int q) const { return min(r.a.M - m_begin(q), r.rows_max); }
    __device__ __forceinline__ const uint8_t* row_at(int q, int, int m) const {
      return r.a.x + (long long)(m_begin(q) + m) * r.a.ldx;
    }
    __device__ __forceinline__ void weights(int item) {
      const int n0 = tile(item) % tiles * S::kTile;
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
      const int t = tile(item), n0 = t % tiles * S::kTile, q = part(item);
      const int m0 = t / tiles * r.rows_max, n_rows = min(r.a.M - m0, r.rows_max);
      auto* mine = held + slot(item) * 16 * kMT * S::kTile;
      for (int i = (int)threadIdx.x; i < n_rows * S::kTile; i += S::kThreads) {
        const int c = i % S::kTile, row = i / S::kTile, n = n0 + c, m = m0 + row;
        float f = st.sum_of(0, c / 16, row / 16, row % 16, c % 16);
        if (q > 0) f += mine[i];
        if (q < r.parts - 1) {
          mine[i] = f;
          continue;
        }
        if (n >= r.a.N) continue;
        if (!(__builtin_fabsf(f) < __builtin_inff())) f = slow_row<kX, kW, kS>(r.a, m, n);
        if (r.a.bias) f += r.a.bias[n];
        store_result(r.a.y, m * r.a.ldy + n, r.a.out, activate(f, r.a.act));
      }
    }
  };
  const int tiles = (r.a.N + S::kTile - 1) / S::kTile;
  const long long all = (long long)((r.a.M + r.rows_max - 1) / r.rows_max) * tiles;
  Policy p{{}, r, (__attribute__((address_space(3))) float*)held,
           (int)(all * blockIdx.x / gridDim.x), (int)(all * (blockIdx.x + 1) / gridDim.x), tiles};
  p.st.lds = (lds_u8*)lds;
  p.st.rings = (lds_u8*)rings;
  p.st.sums = (__attribute__((address_space(3))) float*)sums;
  p.st.K = r.a.K;
  p.st.ldw = (uint32_t)r.a.ldw;
  p.st.inv = 32.0f / (float)r.a.G;
  p.st.run(0, (p.t1 - p.t0) * r.parts, r.len, p);
}

}  // namespace detail
}  // namespace hipgemm
