// The experts of a mixture-of-experts layer for a few tokens:
//
//   k_moe_up    h[p] = weights[p] act(x[t] W13[e][:F]^T) (x[t] W13[e][F:]^T)
//               for each pair p = (token t, its j-th choice), e = ids[p]
//   k_moe_down  o[q][p] = h[p] W2[e]^T over the q-th part of F
//   k_moe_sum   y[t] = sum_j sum_q o[q][t k + j]
//
// What bounds it: each chosen expert's weights, read once for as many of its tokens
// as LDS has room for (going up 37120 / D rows of x, at most 16, or 32 where experts have
// many; going down as many of h, for which F is cut into parts), so the first two
// stream weights past the few rows that
// need them (w4_stream.hpp: Stream), one workgroup per CU, which share the work
// evenly: all tiles of weights of all chosen experts, in order, cut into as many
// pieces as there are workgroups.  Which experts those are, and their pairs, each
// workgroup finds from the ids (at most kMoePairs) by itself, by counting.
//
// The contributions to an output are written apart, by pair and part, and summed
// in their order: no atomics, the same result every time.
//
// h is held as the sum of two bf16 numbers (16 significand bits; one rounding to
// bf16 would leave an error as large as the output's own), of three for fp32
// results (24 bits, its own), and the second kernel multiplies all parts: its matrix
// unit is idle most of the time.  16 bits leave 3e-6 of the results' rms, a
// thousandth of a bf16 result's rounding, 24 bits 2e-7; three parts everywhere
// would cost (us, three / two) 64 tokens, 8 of 128 of 4096 x 1536 int4 297/266, 8 of 64
// of 2048 x 1024 85/64, one token of 2 of 8 of 4096 x 14336 59/53 (e4m3 74/70).
#pragma once

#include "w4_stream.hpp"
#include "w4_vec.hpp"

namespace hipgemm {
namespace detail {

constexpr int kMoePairs = 512;     // of one launch
constexpr int kMoeExperts = 1024;  // two per thread

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
  uint16_t* h;  // pairs x h_parts x F
  float* o;     // parts x pairs x D
  int T, k, E, D, F, G;
  int act, out;
  int h_parts;  // of h: 2, 3
  int parts, part_len;  // k_moe_down: of F
  int waves_k, rows, wave_rows;  // k_moe_vec_*: of a workgroup, of a wave
};

// One value of h, in its parts (one that is infinite, or in bf16, has no rest).
__device__ __forceinline__ void store_h(const MoeArgs& g, int pair, int f, float v) {
  uint16_t* h = g.h + (long long)pair * g.h_parts * g.F + f;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    if (i == g.h_parts) break;
    const __bf16 part = (__bf16)v;
    h[i * g.F] = __builtin_bit_cast(uint16_t, part);
    v -= (float)part;
    if (!(__builtin_fabsf(v) < __builtin_inff())) v = 0.0f;
  }
}

// The pairs by expert: groups of up to rows_max pairs of one expert.
struct MoeGroups {
  uint16_t expert[kMoePairs], begin[kMoePairs], rows[kMoePairs];
  // Pairs, by group (their experts while they are counted).
  __attribute__((aligned(16))) uint16_t list[kMoePairs];
  // By pair (a load of memory at an item's end would wait for the weights ahead).
  float weight[kMoePairs];
};

constexpr int kMoeTables = 7 << 10;
static_assert(sizeof(MoeGroups) <= kMoeTables - 512, "room for the tables");

// Fills t, by all 512 threads; count: LDS of kMoeExperts + 8 ints, free after.
// Returns the number of groups.  A pair's place among its expert's is where the
// counting put it, which may differ between workgroups: nothing depends on the
// order within a group.  Where an expert has several groups, all workgroups have
// to agree on them, and places go by the pairs' order.
__device__ __forceinline__ int moe_groups(const MoeArgs& g, int rows_max, MoeGroups& t,
                                          __attribute__((address_space(3))) int* count) {
  const int tid = (int)threadIdx.x, wave = wave_id(), lane = lane_id();
  const int pairs = g.T * g.k;
  auto* totals = count + kMoeExperts;
  const int id = tid < pairs ? g.ids[tid] : -1;
  const bool on = id >= 0 && id < g.E;
  count[2 * tid] = count[2 * tid + 1] = 0;
  __syncthreads();
  int rank = 0;
  if (on) rank = __hip_atomic_fetch_add(&count[id], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  t.list[tid] = (uint16_t)(on ? id : 0xffff);
  t.weight[tid] = on ? g.weights[tid] : 0.0f;
  __syncthreads();
  // A thread's two experts; both sums at once: pairs above, groups below.
  const int n[2] = {count[2 * tid], count[2 * tid + 1]};
  const int groups[2] = {(n[0] + rows_max - 1) / rows_max, (n[1] + rows_max - 1) / rows_max};
  const int mine = (n[0] + n[1]) << 16 | (groups[0] + groups[1]);
  int sum = mine;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int v = __shfl_up(sum, d, kWave);
    if (lane >= d) sum += v;
  }
  if (lane == kWave - 1) totals[wave] = sum;
  const bool several = __syncthreads_or(groups[0] > 1 || groups[1] > 1);
  if (several && on) {
    rank = 0;
    for (int j = 0; j < 64 * (wave + 1); j += 8) {
      const i32x4 v = *reinterpret_cast<const i32x4*>(t.list + j);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int other = (int)((uint32_t)v[i / 2] >> (16 * (i & 1)) & 0xffffu);
        rank += other == id && j + i < tid;
      }
    }
  }
  int all = 0;
  for (int w = 0; w < 8; ++w) {
    const int v = totals[w];
    if (w < wave) sum += v;
    all += v;
  }
  int before = sum - mine;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int at = before >> 16;
    for (int i = 0; i < groups[x]; ++i) {
      const int q = (before & 0xffff) + i;
      t.expert[q] = (uint16_t)(2 * tid + x);
      t.begin[q] = (uint16_t)(at + i * rows_max);
      t.rows[q] = (uint16_t)min(rows_max, n[x] - i * rows_max);
    }
    count[2 * tid + x] = at;
    before += n[x] << 16 | groups[x];
  }
  __syncthreads();
  if (on) t.list[count[id] + rank] = (uint16_t)tid;
  __syncthreads();
  return all & 0xffff;
}

// This workgroup's share of items.
__device__ __forceinline__ void share(int items, int* first, int* last) {
  *first = (int)((long long)items * blockIdx.x / gridDim.x);
  *last = (int)((long long)items * (blockIdx.x + 1) / gridDim.x);
}

template <int kX, int kW, int kS, int kMode, int kMT, int kWK>
__global__ __launch_bounds__(512) void k_moe_up(MoeArgs g) {
  using S = Stream<kX, kW, kS, kMode, kMT, 1, kWK, kMoeTables>;
  constexpr int kCols = 16 * S::kWN;  // of F, of an item: gate and up rows
  __shared__ __attribute__((aligned(16))) uint8_t lds[S::kXBytes];
  __shared__ __attribute__((aligned(1024))) uint8_t rings[S::kRingBytes];
  __shared__ float sums[S::kSums];
  __shared__ MoeGroups t;
  const int n_groups = moe_groups(g, S::rows_that_fit(g.D), t,
                                  (__attribute__((address_space(3))) int*)(lds_u8*)lds);
  const int tiles = (g.F + kCols - 1) / kCols;

  struct Policy {
    S st;
    const MoeArgs& g;
    const MoeGroups& t;
    int tiles;
    __device__ __forceinline__ int group(int item) const { return item / tiles; }
    __device__ __forceinline__ int k_begin(int) const { return 0; }
    __device__ __forceinline__ int rows(int q) const {
      return __builtin_amdgcn_readfirstlane(t.rows[q]);
    }
    __device__ __forceinline__ int pair(int q, int m) const { return t.list[t.begin[q] + m]; }
    __device__ __forceinline__ const uint8_t* row_at(int q, int, int m) const {
      return g.x + (long long)(__builtin_amdgcn_readfirstlane(pair(q, m)) / g.k) * g.ldx;
    }
    __device__ __forceinline__ void weights(int item) {
      const int q = item / tiles, e = __builtin_amdgcn_readfirstlane(t.expert[q]);
      // (a set past the end: the last columns again, not used)
      const int f0 = min((item - q * tiles) * kCols + 16 * st.set(), g.F - 16);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        st.set_tile(n, g.w13 + e * g.w13_expert + ((long long)n * g.F + f0) * g.w13_row);
        const long long r = (long long)st.scale_tile(n) * g.F + f0 + (lane_id() & 15);
        st.sp[n] = g.s13 + e * g.s13_expert + r * g.s13_row;
        if constexpr (kW == kWInt4Z) st.zp[n] = g.z13 + e * g.z13_expert + r * g.z13_row;
      }
    }
    __device__ __forceinline__ void finish(int item) {
      const int q = item / tiles, f0 = (item - q * tiles) * kCols, n_rows = rows(q);
      // One value per thread and turn: neighbouring columns in neighbouring threads.
      for (int i = (int)threadIdx.x; i < n_rows * kCols; i += S::kThreads) {
        const int c = i % kCols, r = i / kCols, f = f0 + c;
        if (f >= g.F) continue;
        const float a = st.sum_of(c / 16, 0, r / 16, r % 16, c % 16);
        const float b = st.sum_of(c / 16, 1, r / 16, r % 16, c % 16);
        const int p = pair(q, r);
        store_h(g, p, f, activate(a, g.act) * b * t.weight[p]);
      }
    }
  };
  Policy p{{}, g, t, tiles};
  p.st.lds = (lds_u8*)lds;
  p.st.rings = (lds_u8*)rings;
  p.st.sums = (__attribute__((address_space(3))) float*)sums;
  p.st.K = g.D;
  p.st.ldw = (uint32_t)g.w13_row;
  p.st.inv = 32.0f / (float)g.G;
  int first, last;
  share(n_groups * tiles, &first, &last);
  p.st.run(first, last, g.D, p);
}

template <int kW, int kS, int kMode, int kMT, int kWK, int kH>
__global__ __launch_bounds__(512) void k_moe_down(MoeArgs g) {
  using S = Stream<kInBf16, kW, kS, kMode, kMT, kH, kWK, kMoeTables>;
  __shared__ __attribute__((aligned(16))) uint8_t lds[S::kXBytes];
  __shared__ __attribute__((aligned(1024))) uint8_t rings[S::kRingBytes];
  __shared__ float sums[S::kSums];
  __shared__ MoeGroups t;
  const int n_groups = moe_groups(g, S::rows_that_fit(g.part_len), t,
                                  (__attribute__((address_space(3))) int*)(lds_u8*)lds);
  const int tiles = (g.D + S::kTile - 1) / S::kTile;

  struct Policy {
    S st;
    const MoeArgs& g;
    const MoeGroups& t;
    int tiles;
    // Groups here: an expert's rows over a part of F.
    __device__ __forceinline__ int group(int item) const { return item / tiles; }
    __device__ __forceinline__ int k_begin(int item) const {
      return item / tiles % g.parts * g.part_len;
    }
    __device__ __forceinline__ int rows(int q) const {
      return __builtin_amdgcn_readfirstlane(t.rows[q / g.parts]);
    }
    __device__ __forceinline__ int pair(int q, int m) const {
      return t.list[t.begin[q / g.parts] + m];
    }
    __device__ __forceinline__ const uint8_t* row_at(int q, int part, int m) const {
      return reinterpret_cast<const uint8_t*>(
          g.h + ((long long)__builtin_amdgcn_readfirstlane(pair(q, m)) * kH + part) * g.F);
    }
    __device__ __forceinline__ void weights(int item) {
      const int q = item / tiles, e = __builtin_amdgcn_readfirstlane(t.expert[q / g.parts]);
      const int d0 = min((item - q * tiles) * S::kTile + 32 * st.set(), g.D - 32);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        st.set_tile(n, g.w2 + e * g.w2_expert + (long long)(d0 + 16 * n) * g.w2_row);
        const long long r = d0 + 16 * st.scale_tile(n) + (lane_id() & 15);
        st.sp[n] = g.s2 + e * g.s2_expert + r * g.s2_row;
        if constexpr (kW == kWInt4Z) st.zp[n] = g.z2 + e * g.z2_expert + r * g.z2_row;
      }
    }
    __device__ __forceinline__ void finish(int item) {
      const int q = item / tiles, d0 = (item - q * tiles) * S::kTile, n_rows = rows(q);
      for (int i = (int)threadIdx.x; i < n_rows * S::kTile; i += S::kThreads) {
        const int c = i % S::kTile, r = i / S::kTile, d = d0 + c;
        if (d >= g.D) continue;
        g.o[((long long)(q % g.parts) * (g.T * g.k) + pair(q, r)) * g.D + d] =
            st.sum_of(c / 32, c / 16 % 2, r / 16, r % 16, c % 16);
      }
    }
  };
  Policy p{{}, g, t, tiles};
  p.st.lds = (lds_u8*)lds;
  p.st.rings = (lds_u8*)rings;
  p.st.sums = (__attribute__((address_space(3))) float*)sums;
  p.st.K = g.F;
  p.st.ldw = (uint32_t)g.w2_row;
  p.st.inv = 32.0f / (float)g.G;
  int first, last;
  share(n_groups * g.parts * tiles, &first, &last);
  p.st.run(first, last, g.part_len, p);
}

}  // namespace detail
}  // namespace hipgemm
