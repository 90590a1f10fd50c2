// The experts of a mixture-of-experts layer for a few tokens, in two kernels:
//
//   k_moe_up    h[p] = weights[p] act(x[t] W13[e][:F]^T) (x[t] W13[e][F:]^T)
//               for each pair p = (token t, its j-th choice), e = ids[p]
//   k_moe_down  y[t] = sum_j h[t k + j] W2[e]^T
//
// What bounds it: each chosen expert's weights are read once, whatever the
// number of its tokens, so both stream weights past the few rows that need them
// (w4_stream.hpp: Stream).
//
// k_moe_up: a workgroup takes an expert and 16 of its F columns, gate and up,
// and deals K to its waves.  The experts in question are found from the ids by
// the workgroup itself (a ballot over at most kMoePairs ids): blockIdx.y names a
// pair, which does the work if it is the first of its expert, or, where there are
// more pairs than experts, the expert.  What it found goes to a table for the
// second kernel.
//
// k_moe_down: a workgroup takes 16 columns of y for all chosen experts, dealt to
// its waves by expert and part of K, so that all contributions to an output meet
// in one workgroup's LDS, by pair, and are summed in the order of j: no atomics,
// the same result every time.
//
// h is held as the sum of two bf16 numbers (16 significand bits; one rounding to
// bf16 would leave an error as large as the output's own), and the second
// kernel multiplies both parts: its matrix unit is idle most of the time.
#pragma once

#include "w4_stream.hpp"
#include "w4_vec.hpp"

namespace hipgemm {
namespace detail {

constexpr int kMoePairs = 512;  // of one launch

// Strides in bytes, but ldy in elements.
struct MoeArgs {
  const uint8_t* x;
  const int* ids;
  const float* weights;
  const uint8_t *w13, *s13, *z13, *w2, *s2, *z2;
  long long ldx, ldy;
  long long w13_row, w13_expert, s13_row, s13_expert, z13_row, z13_expert;
  long long w2_row, w2_expert, s2_row, s2_expert, z2_row, z2_expert;
  uint8_t* y;
  uint16_t* h;  // pairs x 2 x F: high parts, low parts
  int* table;   // per slot: pairs, expert, kMoePairs of list
  int T, k, E, D, F, G13, G2;
  int act, out;
  int by_pair;    // slots are pairs (else experts)
  int slots;
  int max_parts;  // k_moe_down: parts of K at most
};

constexpr int kMoeTable = 2 + kMoePairs;

template <int kX, int kW, int kS, int kMode, int kMT>
__global__ __launch_bounds__(512) void k_moe_up(MoeArgs g) {
  const int wave = wave_id(), lane = lane_id(), tid = (int)threadIdx.x;
  const int slot = (int)blockIdx.y, f0 = (int)blockIdx.x * 16;
  __shared__ uint64_t match[8];
  __shared__ int list[kMoePairs];
  const int pairs = g.T * g.k;
  const int e = g.by_pair ? g.ids[slot] : slot;
  const bool valid = e >= 0 && e < g.E;
  const bool mine = valid && tid < pairs && g.ids[tid] == e;
  const uint64_t here = __builtin_amdgcn_ballot_w64(mine);
  if (lane == 0) match[wave] = here;
  __syncthreads();
  int count = 0, before = 0, first = kMoePairs;
#pragma unroll
  for (int w = 7; w >= 0; --w) {
    const uint64_t m = match[w];
    count += __builtin_popcountll(m);
    if (w < wave) before += __builtin_popcountll(m);
    if (m) first = 64 * w + __builtin_ctzll(m);
  }
  if (g.by_pair && first != slot) count = 0;
  if (mine) list[before + __builtin_popcountll(here & ((1ull << lane) - 1ull))] = tid;
  __syncthreads();
  if (blockIdx.x == 0) {
    int* t = g.table + (long long)slot * kMoeTable;
    if (tid == 0) {
      t[0] = count;
      t[1] = e;
    }
    if (tid < count) t[2 + tid] = list[tid];
  }
  if (count == 0) return;

  Stream<kX, kW, kS, kMode, 2, kMT, false> st;
  st.K = g.D;
  st.lo = 0;
  st.inv = 32.0f / (float)g.G13;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const long long r = n * g.F + f0 + (lane & 15);
    st.w[n] = g.w13 + e * g.w13_expert + r * g.w13_row;
    st.s[n] = g.s13 + e * g.s13_expert + r * g.s13_row;
    st.z[n] = g.z13 ? g.z13 + e * g.z13_expert + r * g.z13_row : nullptr;
  }
  __shared__ float part[8][2][kMT][kWave * 4];
  for (int m0 = 0; m0 < count; m0 += 16 * kMT) {
#pragma unroll
    for (int m = 0; m < kMT; ++m) {
      st.x[m] = g.x + (long long)(list[min(m0 + 16 * m + (lane & 15), count - 1)] / g.k) * g.ldx;
      st.acc[0][m] = st.acc[1][m] = f32x4{};
    }
    st.run(wave, st.pairs(), 8);
    if (m0) __syncthreads();
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int m = 0; m < kMT; ++m)
        *reinterpret_cast<f32x4*>(&part[wave][n][m][4 * lane]) = st.acc[n][m];
    __syncthreads();
    // One value per thread: 16 columns of a row in neighbouring threads.
    for (int t = tid; t < 256 * kMT; t += 512) {
      const int m = t >> 8, row = (t >> 4) & 15, col = t & 15;
      const int at = 4 * (16 * (row >> 2) + col) + (row & 3);
      float a = 0.0f, b = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        a += part[w][0][m][at];
        b += part[w][1][m][at];
      }
      const int r = m0 + 16 * m + row;
      if (r >= count) continue;
      const int f = f0 + col;
      if constexpr (kW == kWE4M3) {
        const uint8_t* s = g.s13 + e * g.s13_expert;
        a *= *reinterpret_cast<const float*>(s + f * g.s13_row);
        b *= *reinterpret_cast<const float*>(s + (g.F + f) * g.s13_row);
      }
      const int p = list[r];
      const float v = activate(a, g.act) * b * g.weights[p];
      const __bf16 hi = (__bf16)v;
      const float rest = v - (float)hi;
      // (an infinite h has no rest)
      const __bf16 lo = (__bf16)(rest == rest ? rest : 0.0f);
      uint16_t* h = g.h + (long long)p * 2 * g.F + f;
      h[0] = __builtin_bit_cast(uint16_t, hi);
      h[g.F] = __builtin_bit_cast(uint16_t, lo);
    }
  }
}

template <int kW, int kS, int kMode>
__global__ __launch_bounds__(512) void k_moe_down(MoeArgs g) {
  const int wave = wave_id(), lane = lane_id(), tid = (int)threadIdx.x;
  const int waves = (int)blockDim.x / kWave;
  const int d0 = (int)blockIdx.x * 16;
  const int pairs = g.T * g.k;
  extern __shared__ float sums[];  // max_parts x pairs x 16
  __shared__ uint64_t have[8];
  __shared__ int active[kMoePairs];
  // The slots that have pairs, in order.
  const bool on = tid < g.slots && g.table[(long long)tid * kMoeTable] > 0;
  const uint64_t here = __builtin_amdgcn_ballot_w64(on);
  if (wave < 8 && lane == 0) have[wave] = here;
  for (int i = tid; i < g.max_parts * pairs * 4; i += (int)blockDim.x)
    reinterpret_cast<f32x4*>(sums)[i] = f32x4{};
  __syncthreads();
  int n_active = 0, before = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const uint64_t m = w < waves ? have[w] : 0ull;
    n_active += __builtin_popcountll(m);
    if (w < wave) before += __builtin_popcountll(m);
  }
  if (on) active[before + __builtin_popcountll(here & ((1ull << lane) - 1ull))] = tid;
  __syncthreads();

  Stream<kInBf16, kW, kS, kMode, 1, 1, true> st;
  st.K = g.F;
  st.lo = 2ll * g.F;
  st.inv = 32.0f / (float)g.G2;
  // Parts of K: as many as leave every wave something to do.
  const int steps = st.pairs();
  int parts = 1;
  while (2 * parts <= g.max_parts && 2 * parts <= steps && n_active * parts < waves) parts *= 2;
  for (int item = wave; item < n_active * parts; item += waves) {
    const int part = item % parts;
    const int* t = g.table + (long long)__builtin_amdgcn_readfirstlane(active[item / parts]) * kMoeTable;
    const int count = t[0], e = t[1];
    const long long r = d0 + (lane & 15);
    st.w[0] = g.w2 + e * g.w2_expert + r * g.w2_row;
    st.s[0] = g.s2 + e * g.s2_expert + r * g.s2_row;
    st.z[0] = g.z2 ? g.z2 + e * g.z2_expert + r * g.z2_row : nullptr;
    float row_scale = 1.0f;
    if constexpr (kW == kWE4M3) row_scale = *reinterpret_cast<const float*>(st.s[0]);
    for (int m0 = 0; m0 < count; m0 += 16) {
      st.x[0] = reinterpret_cast<const uint8_t*>(
          g.h + (long long)t[2 + min(m0 + (lane & 15), count - 1)] * 2 * g.F);
      st.acc[0][0] = f32x4{};
      st.run(part * steps / parts, (part + 1) * steps / parts, 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = m0 + 4 * (lane >> 4) + i;
        if (row < count)
          sums[(part * pairs + t[2 + row]) * 16 + (lane & 15)] = st.acc[0][0][i] * row_scale;
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < g.T * 16; i += (int)blockDim.x) {
    const int tok = i >> 4, col = i & 15;
    float v = 0.0f;
    for (int j = 0; j < g.k; ++j)
      for (int q = 0; q < parts; ++q) v += sums[(q * pairs + tok * g.k + j) * 16 + col];
    store_result(g.y, tok * g.ldy + d0 + col, g.out, v);
  }
}

}  // namespace detail
}  // namespace hipgemm
