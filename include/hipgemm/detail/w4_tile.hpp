// Products of 5 rows of 16-bit activations and more with 4-bit weights, by MFMA.  A
// wave multiplies 16 kMT rows of x by 16 kNT of weights (W4Wave), 128 of K at a
// time: x (256 bytes of a row) and weights (64 bytes) come by DMA into stages of
// LDS, weights are decoded in registers on their way to the matrix unit.
//
// k_w4_split, some rows: what bounds it is the weights' and x's way into a CU, and
// for few steps the first loads' latency.  Four waves take every fourth step of
// one tile each, with stages of their own, so nobody waits for anybody until the
// sums are added; up to 160 KiB of stages are on their way.  bf16, us in a graph:
// 16 x 14336 x 4096 fp4 in groups of 32 16.1 (2.0 TB/s), 16 x 28672 x 8192 int4 52,
// 64 x 14336 x 4096 int4 24, 37 x 5000 x 3584 int4 in groups of 64 19.  (With all of
// x of a group in LDS and the weights streaming past it the same took 18.6, 53, 104,
// 35: x came in again for every 32 columns.)
//
// k_w4_tile, many rows: bound by the matrix unit and by what surrounds it.  Tiles of
// 128 x 128 by four waves, 64 x 64 each, two stages of 40 KiB that they share, two
// workgroups to a CU, so that one's arithmetic hides the other's waits.  2048 x 14336
// x 4096 int4, group 128, bf16: 297 us, 810 TFLOP/s (628 by k_w4_split).
//
// Per wave of 64 x 64 and step there are 64 MFMAs of 16 cycles each; the decoding
// takes 9 instructions per 8 weights and lane (16 x 9), int4 with one scale per step
// and row one FMA per accumulator (64): all told about as many issue slots as the
// matrix unit takes, so neither may grow.  Hence:
//   * int4 codes are decoded in their own order (decode.hpp): reordering activations
//     would cost as much as the decoding (16 operands against 16).
//   * the zero point's share, -z sum(x), is the accumulator that a step's MFMAs
//     start from: without zero points it is the same for all columns.
// Scales as in w4_stream.hpp (kCoarse, kFine, kInline), loaded with the stage by the
// lanes that need them.
//
// A row of x's chunk c (16 bytes) lies at slot c ^ x_slot(row), one of weights (16
// bytes, four to a row) at slot c ^ (row / 2 % 4).  A read of 16 bytes per lane takes
// lanes 0-3, 12-15, 20-27 together, and so on: eight rows of one chunk and the
// other eight of the next or the fourth from it, which have to lie on all banks.
// (With c ^ (row % 16) 43% of the LDS cycles were conflicts.)
#pragma once

#include "layout.hpp"
#include "w4_stream.hpp"
#include "w4_vec.hpp"

namespace hipgemm {
namespace detail {

constexpr int kW4TileM = 128, kW4TileN = 128, kW4TileK = 128;

// (rows 0-3, 12-15 have slots 0-7, the others 8-15: xor 1 or 4 stays in these)
__device__ __forceinline__ int x_slot(int row) { return (row + 4) & 15; }

// Sums that came out infinite or NaN, by the definition, weight by weight: the sums
// before the scale can overflow for an x near the largest, and an infinite one makes
// NaN of zero points, where the definition has an infinity or a number.  All of the
// wave's lanes take their bad sums (row m, column n) one after the other, each a
// share of K in units of 32.  A row that holds a NaN has nothing else to give, so
// its lanes are done together: 2048 rows of NaN by 14336 x 4096 take 1.0 ms, with an
// infinity in each row, which can give a number, 36 ms (0.3 without).
template <int kX, int kW, int kS>
__device__ __forceinline__ float by_definition(const W4Args& g, int m, int n, bool bad, float v) {
  int lane = lane_id();
  asm volatile("" : "+v"(lane));  // (nothing of this is to be held during the products)
  const float inv = 32.0f / (float)g.G;
  uint64_t todo = __builtin_amdgcn_ballot_w64(bad);
  while (todo) {
    const int first = __builtin_ctzll(todo);
    const int row = __builtin_amdgcn_readlane(m, first);
    const uint8_t* x = g.x + row * g.ldx;
    uint64_t mine = __builtin_amdgcn_ballot_w64(bad && m == row);
    todo &= ~mine;
    bool nan = false;
#pragma unroll 1
    for (int k = 8 * lane; k < g.K; k += 8 * kWave) {
      const i32x4 a = *reinterpret_cast<const i32x4*>(x + 2ll * k);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2 f = unpack2<kX>((uint32_t)a[i]);
        nan |= f[0] != f[0] || f[1] != f[1];
      }
    }
    if (__builtin_amdgcn_ballot_w64(nan)) {
      if (bad && m == row) v = __builtin_nanf("");
      continue;
    }
    while (mine) {
      const int to = __builtin_ctzll(mine), col = __builtin_amdgcn_readlane(n, to);
      mine &= mine - 1;
      const uint8_t* w = g.w + col * g.ldw;
      float sum = 0.0f;
#pragma unroll 1
      for (int u = lane; u < g.K / 32; u += kWave) {
        const int grp = group_of(u, inv);
        const float s = scale_at<kS>(g.s + col * g.lds, grp);
        const float z = g.z ? (float)g.z[col * g.ldz + grp] : 8.0f;
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          const uint32_t q = *reinterpret_cast<const uint32_t*>(w + 16ll * u + 4 * j);
          const i32x4 a = *reinterpret_cast<const i32x4*>(x + 64ll * u + 16 * j);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x2 f = unpack2<kX>((uint32_t)a[i]);
            sum = __builtin_fmaf(f[0], s * code_value<kW>(q >> (8 * i) & 15u, z), sum);
            sum = __builtin_fmaf(f[1], s * code_value<kW>(q >> (8 * i + 4) & 15u, z), sum);
          }
        }
      }
#pragma unroll
      for (int d = 1; d < kWave; d *= 2) sum += __shfl_xor(sum, d, kWave);
      if (lane == to) v = sum;
    }
  }
  return v;
}

// What a wave multiplies: 16 kMT rows of x by 16 kNT of weights, 128 of K.
template <int kX, int kW, int kS, int kMode, int kMT, int kNT>
struct W4Wave {
  static constexpr bool kZ = kW == kWInt4Z;
  f32x4 acc[kNT][kMT];  // [n][m]

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int m = 0; m < kMT; ++m) acc[n][m] = f32x4{};
  }

  // Reads of LDS in assembly, with their waits (w4_stream.hpp: read_x): 16 bytes
  // each of rows r, 16 + r, ...
  __device__ __forceinline__ static void read_x(const lds_u8* p, i32x4 (&v)[kMT]) {
    if constexpr (kMT == 1)
      asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v[0]) : "v"(p) : "memory");
    else if constexpr (kMT == 2)
      asm volatile(
          "ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:4096\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(v[0]), "=&v"(v[1])
          : "v"(p)
          : "memory");
    else if constexpr (kMT == 3)
      asm volatile(
          "ds_read_b128 %0, %3\n\tds_read_b128 %1, %3 offset:4096\n\t"
          "ds_read_b128 %2, %3 offset:8192\n\ts_waitcnt lgkmcnt(0)"
          : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2])
          : "v"(p)
          : "memory");
    else
      asm volatile(
          "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:4096\n\t"
          "ds_read_b128 %2, %4 offset:8192\n\tds_read_b128 %3, %4 offset:12288\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
          : "v"(p)
          : "memory");
  }
  __device__ __forceinline__ static void read_w(const lds_u8* p, i32x4 (&v)[kNT]) {
    if constexpr (kNT == 2)
      asm volatile(
          "ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:1024\n\ts_waitcnt lgkmcnt(0)"
          : "=&v"(v[0]), "=&v"(v[1])
          : "v"(p)
          : "memory");
    else
      asm volatile(
          "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:1024\n\t"
          "ds_read_b128 %2, %4 offset:2048\n\tds_read_b128 %3, %4 offset:3072\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
          : "v"(p)
          : "memory");
  }

  // x and w: the wave's first rows in a stage;  s, z: raw scales and zero points of
  // rows 16 n + r.
  __device__ __forceinline__ void multiply(const lds_u8* x, const lds_u8* w_, const uint32_t (&s)[kNT],
                                           const uint32_t (&z)[kNT]) {
    i32x4 q[kNT];
    const int r = lane_id() & 15, gq = lane_id() >> 4;
    read_w(w_ + r * 64 + 16 * (gq ^ ((r >> 1) & 3)), q);
    const lds_u8* ap = x + r * 256;
    const int one = (int)kOnes2<kX>;
    const i32x4 ones{one, one, one, one};
    if constexpr (kMode == kFine) {
      // MFMA j: the lane's k = 32 j + 8 gq, one scale for all of it.
      uint32_t w[kNT][4], s4[kNT][4], z4[kNT][4];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[n][i] = (uint32_t)q[n][i];
        transpose4(w[n]);
        spread4(s[n], s4[n]);
        if constexpr (kZ) spread4(z[n], z4[n]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        i32x4 a[kMT];
        read_x(ap + 16 * ((4 * j + gq) ^ x_slot(r)), a);
        f32x4 xs[kMT];
        if constexpr (is_int4(kW)) {
#pragma unroll
          for (int m = 0; m < kMT; ++m) {
            xs[m] = mfma_16x16x32<kX>(a[m], ones, f32x4{});
            if constexpr (!kZ) xs[m] *= -8.0f;
          }
        }
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          const i32x4 b = decode8<kX, kW>(w[n][j], 0u, 1.0f);
          const float c = scale_of<kS>(s4[n][j]);
#pragma unroll
          for (int m = 0; m < kMT; ++m) {
            f32x4 p = f32x4{};
            if constexpr (kZ) p = xs[m] * -(float)z4[n][j];
            else if constexpr (is_int4(kW)) p = xs[m];
            p = mfma_16x16x32<kX>(a[m], b, p);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][m][e] = __builtin_fmaf(c, p[e], acc[n][m][e]);
          }
        }
      }
    } else {
      // MFMA j: the lane's k = 32 gq + 8 j.  One accumulator after the other: four
      // MFMAs that depend on each other would wait for each other.
      i32x4 a[4][kMT];
#pragma unroll
      for (int j = 0; j < 4; ++j) read_x(ap + 16 * ((4 * gq + j) ^ x_slot(r)), a[j]);
      f32x4 xs[kMT];
      if constexpr (is_int4(kW)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int m = 0; m < kMT; ++m)
            xs[m] = mfma_16x16x32<kX>(a[j][m], ones, j == 0 ? f32x4{} : xs[m]);
        if constexpr (!kZ) {
#pragma unroll
          for (int m = 0; m < kMT; ++m) xs[m] *= -8.0f;
        }
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const float c = scale_of<kS>(s[n]);
        f32x4 p[kMT];
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          if constexpr (kMode == kInline) p[m] = acc[n][m];
          else if constexpr (kZ) p[m] = xs[m] * -(float)z[n];
          else if constexpr (is_int4(kW)) p[m] = xs[m];
          else p[m] = f32x4{};
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const i32x4 b = decode8<kX, kW>((uint32_t)q[n][j], 0u, kMode == kInline ? c : 1.0f);
#pragma unroll
          for (int m = 0; m < kMT; ++m) p[m] = mfma_16x16x32<kX>(a[j][m], b, p[m]);
        }
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          if constexpr (kMode == kInline) {
            acc[n][m] = p[m];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][m][e] = __builtin_fmaf(c, p[m][e], acc[n][m][e]);
          }
        }
      }
    }
  }
};

// The loads of W4Wave's scales.
template <int kW, int kS, int kMode, int kNT>
struct W4Scales {
  static constexpr bool kZ = kW == kWInt4Z;
  static constexpr int kLoads = kZ ? 2 * kNT : kNT;
  const uint8_t *s, *z;
  uint32_t row[kNT];
  int K;
  float inv;

  // Rows n0 + 16 n + r.
  __device__ __forceinline__ void set(const W4Args& g, int n0) {
    n0 = min(n0, g.N - 1);
    s = g.s + (long long)n0 * g.lds;
    z = kZ ? g.z + (long long)n0 * g.ldz : nullptr;
#pragma unroll
    for (int n = 0; n < kNT; ++n)
      row[n] = (uint32_t)min(16 * n + (lane_id() & 15), g.N - 1 - n0) * (uint32_t)g.ldz;
    K = g.K;
    inv = 32.0f / (float)g.G;
  }
  __device__ __forceinline__ void load(int k, uint32_t (&sv)[kNT], uint32_t (&zv)[kNT]) const {
    const int own = kMode == kCoarse ? k : k + 32 * (lane_id() >> 4);
    const uint32_t at = (uint32_t)group_of(min(own, K - 32) >> 5, inv);
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      sv[n] = scale_raw<kS>(s, row[n] + at);
      if constexpr (kZ) zv[n] = z[row[n] + at];
    }
  }
};

// Rows row .. + 3 of a column; returns whether any of the sums is infinite or NaN.
__device__ __forceinline__ bool w4_store(const W4Args& g, int row, int col, const f32x4& v) {
  if (col >= g.N) return false;
  const float b = g.bias ? g.bias[col] : 0.0f;
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (row + e >= g.M) break;
    float f = v[e];
    odd |= !(__builtin_fabsf(f) < __builtin_inff());
    if (g.bias) f += b;
    store_result(g.y, (row + e) * g.ldy + col, g.out, activate(f, g.act));
  }
  return odd;
}
// Those again, by all lanes of a wave.  (Within the loop that stores the others this
// cost the calls that have none 0.4 us of 16 and 19, and 6 % of 2048 rows.)
template <int kX, int kW, int kS>
__device__ __forceinline__ void w4_store_odd(const W4Args& g, int row, int col, const f32x4& v) {
#pragma unroll 1
  for (int e = 0; e < 4; ++e) {
    float f = e == 0 ? v[0] : e == 1 ? v[1] : e == 2 ? v[2] : v[3];
    const bool bad = col < g.N && row + e < g.M && !(__builtin_fabsf(f) < __builtin_inff());
    f = by_definition<kX, kW, kS>(g, row + e, col, bad, f);
    if (!bad) continue;
    if (g.bias) f += g.bias[col];
    store_result(g.y, (row + e) * g.ldy + col, g.out, activate(f, g.act));
  }
}

template <int kX, int kW, int kS, int kMode>
__global__ __launch_bounds__(256, 2) void k_w4_tile(W4Args g) {
  constexpr int kStageA = kW4TileM * 256, kStageB = kW4TileN * 64;
  constexpr int kStage = kStageA + kStageB;
  __shared__ __attribute__((aligned(1024))) uint8_t lds_[2 * kStage];
  lds_u8* lds = (lds_u8*)lds_;
  const int wave = wave_id(), lane = lane_id();
  const int wm = wave & 1, wn = wave >> 1;

  const int tiles_m = (g.M + kW4TileM - 1) / kW4TileM, tiles_n = (g.N + kW4TileN - 1) / kW4TileN;
  const TileWalk walk = tile_walk((int)blockIdx.x, (int)gridDim.x, tiles_m * tiles_n);
  const uint32_t ldx = (uint32_t)g.ldx, ldw = (uint32_t)g.ldw;
  const int steps = (g.K + kW4TileK - 1) / kW4TileK;

  for (int tile = walk.first; tile < walk.end; tile += walk.stride) {
    const TileCoord tc = grouped_tile_u(tile, tiles_m, tiles_n, 8);
    const int m0 = tc.m * kW4TileM, n0 = tc.n * kW4TileN;
    const auto xb = make_rsrc(g.x + (long long)m0 * g.ldx, (uint32_t)min(g.M - m0, kW4TileM) * ldx);
    const auto wb = make_rsrc(g.w + (long long)n0 * g.ldw, (uint32_t)min(g.N - n0, kW4TileN) * ldw);
    // DMA lanes: x, instruction i (of 32, 8 per wave): rows 4 i .. + 3, lane l row l
    // / 16, slot l % 16;  weights, instruction i (of 8, 2 per wave): rows 16 i .. +
    // 15, lane l row l / 4, slot l % 4.
    auto dma = [&](int k, lds_u8* to) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = 4 * (8 * wave + i) + (lane >> 4);
        const int c = (lane & 15) ^ x_slot(row);
        const int kc = k + 8 * c;
        dma16(xb, to + 1024 * (8 * wave + i), kc < g.K ? (uint32_t)row * ldx + 2 * kc : kOobOffset, 0);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 16 * (2 * wave + i) + (lane >> 2);
        const int c = (lane & 3) ^ ((row >> 1) & 3);
        const int kc = k + 32 * c;
        dma16(wb, to + kStageA + 1024 * (2 * wave + i),
              kc < g.K ? (uint32_t)row * ldw + (kc >> 1) : kOobOffset, 0);
      }
    };
    W4Scales<kW, kS, kMode, 4> sc;
    sc.set(g, n0 + 64 * wn);
    constexpr int kLoads = 10 + W4Scales<kW, kS, kMode, 4>::kLoads;
    W4Wave<kX, kW, kS, kMode, 4, 4> wv;
    wv.clear();
    const int xo = 64 * wm * 256, wo = kStageA + 64 * wn * 64;

    // Step t in stage t % 2; the next step's loads go out before it is waited for.
    uint32_t s[2][4], z[2][4];
    dma(0, lds);
    sc.load(0, s[0], z[0]);
    for (int t = 0; t < steps; t += 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (t + u >= steps) break;
        compiler_fence();
        sched_fence();
        dma((t + u + 1) * kW4TileK, lds + (1 - u) * kStage);  // (past K: zeros)
        sc.load((t + u + 1) * kW4TileK, s[1 - u], z[1 - u]);
        wait_vmcnt<kLoads>();
        barrier();
        wv.multiply(lds + u * kStage + xo, lds + u * kStage + wo, s[u], z[u]);
        wait_lgkmcnt<0>();
        barrier();
      }
    }
    // (the last step's zeros have to land before the stages are used again)
    wait_vmcnt<0>();
    barrier();

    // Each wave's sums through its quarter of the stages, from columns in lanes'
    // registers to whole lines of a row.
    auto sum = (__attribute__((address_space(3))) f32x4*)lds + wave * (2 * kStage / 64);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int m = 0; m < 4; ++m) sum[(n * 4 + m) * kWave + lane] = wv.acc[n][m];
    auto at = [&](int i) {  // rows 4 i .. + 3, column of the lane
      return sum[((lane >> 4) * 4 + (i >> 2)) * kWave + (i & 3) * 16 + (lane & 15)];
    };
    bool odd = false;
#pragma unroll 1
    for (int i = 0; i < 16; ++i) odd |= w4_store(g, m0 + 64 * wm + 4 * i, n0 + 64 * wn + lane, at(i));
    if (__builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll 1
      for (int i = 0; i < 16; ++i)
        w4_store_odd<kX, kW, kS>(g, m0 + 64 * wm + 4 * i, n0 + 64 * wn + lane, at(i));
    }
    barrier();
  }
}

// Some rows: tiles of 16 kMT x 16 kNT, of whose K the four waves take every fourth 128
// each, with stages of their own and no barrier until their sums are added.
template <int kMT, int kNT>
constexpr int kW4SplitStages = (40 << 10) / (kMT * 4096 + kNT * 1024) > 4
                                   ? 4
                                   : (40 << 10) / (kMT * 4096 + kNT * 1024);

template <int kX, int kW, int kS, int kMode, int kMT, int kNT>
__global__ __launch_bounds__(256, 1) void k_w4_split(W4Args g) {
  constexpr int kStageA = kMT * 4096, kStage = kStageA + kNT * 1024, kStages = kW4SplitStages<kMT, kNT>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds_[4 * kStages * kStage];
  const int wave = wave_id(), lane = lane_id();
  lds_u8* lds = (lds_u8*)lds_ + wave * (kStages * kStage);
  const int r = lane & 15;
  const int tiles_m = (g.M + 16 * kMT - 1) / (16 * kMT), tiles_n = (g.N + 16 * kNT - 1) / (16 * kNT);
  const TileWalk walk = tile_walk((int)blockIdx.x, (int)gridDim.x, tiles_m * tiles_n);
  const uint32_t ldx = (uint32_t)g.ldx, ldw = (uint32_t)g.ldw;
  const int steps = ((g.K + 127) / 128 + 3 - wave) / 4;

  for (int tile = walk.first; tile < walk.end; tile += walk.stride) {
    const int m0 = tile % tiles_m * (16 * kMT), n0 = tile / tiles_m * (16 * kNT);
    const auto xb = make_rsrc(g.x + (long long)m0 * g.ldx, (uint32_t)min(g.M - m0, 16 * kMT) * ldx);
    const auto wb = make_rsrc(g.w + (long long)n0 * g.ldw, (uint32_t)min(g.N - n0, 16 * kNT) * ldw);
    auto dma = [&](int k, lds_u8* to) {
#pragma unroll
      for (int i = 0; i < 4 * kMT; ++i) {
        const int row = 4 * i + (lane >> 4);
        const int kc = k + 8 * ((lane & 15) ^ x_slot(row));
        dma16(xb, to + 1024 * i, kc < g.K ? (uint32_t)row * ldx + 2 * kc : kOobOffset, 0);
      }
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        const int row = 16 * i + (lane >> 2);
        const int kc = k + 32 * ((lane & 3) ^ ((row >> 1) & 3));
        dma16_nt(wb, to + kStageA + 1024 * i, kc < g.K ? (uint32_t)row * ldw + (kc >> 1) : kOobOffset, 0);
      }
    };
    W4Scales<kW, kS, kMode, kNT> sc;
    sc.set(g, n0);
    constexpr int kLoads = 4 * kMT + kNT + W4Scales<kW, kS, kMode, kNT>::kLoads;
    W4Wave<kX, kW, kS, kMode, kMT, kNT> wv;
    wv.clear();

    // Step t of this wave in stage t % kStages, kStages - 1 of them ahead.
    uint32_t s[kStages][kNT], z[kStages][kNT];
    auto load = [&](int t, int u) __attribute__((always_inline)) {
      compiler_fence();
      sched_fence();
      const int k = 512 * t + 128 * wave;
      dma(k, lds + u * kStage);  // (past K: zeros)
      sc.load(k, s[u], z[u]);
    };
#pragma unroll
    for (int u = 0; u < kStages - 1; ++u) load(u, u);
    for (int t = 0; t < steps; t += kStages) {
#pragma unroll
      for (int u = 0; u < kStages; ++u) {
        if (t + u >= steps) break;
        load(t + u + kStages - 1, (u + kStages - 1) % kStages);
        wait_vmcnt<(kStages - 1) * kLoads>();
        compiler_fence();
        sched_fence();
        wv.multiply(lds + u * kStage, lds + u * kStage + kStageA, s[u], z[u]);
      }
    }
    // The waves' sums, added in their order.
    wait_vmcnt<0>();
    auto sum = (__attribute__((address_space(3))) f32x4*)(lds_u8*)lds_;
    constexpr int kPer = kStages * kStage / 16;
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int m = 0; m < kMT; ++m) sum[wave * kPer + (n * kMT + m) * kWave + lane] = wv.acc[n][m];
    __syncthreads();
    // (16 x 16 at a time: rows 4 gq .. + 3 of column r in a lane)
    auto at = [&](int i) {
      f32x4 v = sum[i * kWave + lane];
#pragma unroll
      for (int w = 1; w < 4; ++w) v += sum[w * kPer + i * kWave + lane];
      return v;
    };
    bool odd = false;
#pragma unroll 1
    for (int i = wave; i < kNT * kMT; i += 4)
      odd |= w4_store(g, m0 + 16 * (i % kMT) + 4 * (lane >> 4), n0 + 16 * (i / kMT) + r, at(i));
    if (__builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll 1
      for (int i = wave; i < kNT * kMT; i += 4)
        w4_store_odd<kX, kW, kS>(g, m0 + 16 * (i % kMT) + 4 * (lane >> 4), n0 + 16 * (i / kMT) + r,
                                 at(i));
    }
    __syncthreads();
  }
}

}  // namespace detail
}  // namespace hipgemm
