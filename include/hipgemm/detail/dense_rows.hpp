// Products of a few rows of 16-bit activations with 16-bit weights: the forward pass of
// dense.hpp for single tokens and small batches (up to 64 rows), where the weights' bytes
// are all that counts.
//
// A workgroup has kRN rows of the weights (gated: half gate rows, half the up rows of
// the same columns) and all rows of x; its four waves take turns over K, a step of 64
// elements each: whole 128-byte lines, 512 bytes of a row between them.  Every wave
// brings its own steps, kRN rows of weights and 16 kMT rows of x, into its own ring of LDS by
// DMA, as many ahead as its share of the LDS holds, and waits for nobody until its sums are
// done: no barrier in the loop.  Two workgroups of a CU have half of the LDS each, so that
// one's end and start hide behind the other's loads (gated 1 x 14336 x 4096: 40.6 us = 5.8 TB/s
// for 50.7 with one of twice the ring; 16 x 4096 x 14336 25.3 for 26.1).  v_mfma_f32_16x16x32, weights as the first operand, so
// that a lane has four neighbouring columns of one row of x.  At the end the waves' sums
// meet in LDS, are added in order and go through the epilogue of dense.hpp one by one; with
// K-slices (gridDim.y) they go to `partial` instead, for k_dense_reduce.
//
// x is read again by every workgroup, from the L2: kMT times the weights' bytes at most.
// kRN = 16 rows of weights leave every CU some of the usual matrices (1 x 4096 x 4096 8.6 us, with
// 32 11.2, with 64 13.5; 16 x 4096 x 14336 25 / 33 / 49), and lose little where there are
// plenty (gated 1 x 14336 x 4096: 40.6 / 41.2 / 42.8; 32 rows of it 59 / 49 / 50).
#pragma once

#include "dense.hpp"

namespace hipgemm {
namespace detail {

template <int kMT>
struct CfgRows {
  static constexpr int kWaves = 4, kRN = 16;  // rows of weights
  static constexpr int kStage = (kRN + 16 * kMT) * 128;
  static constexpr int kDma = (kRN + 16 * kMT) / 8;
  static constexpr int kRing = 20 * 1024 / kStage;
  static constexpr int kSums = kRN * 16 * kMT * 4;        // of a wave
  static constexpr int kWaveLds = kRing * kStage > kSums ? kRing * kStage : kSums;
  static constexpr int kLdsBytes = kWaves * kWaveLds;
  static_assert(kRing >= 2 && kLdsBytes <= 80 * 1024, "two workgroups of a CU");
  static_assert((kRing - 1) * kDma < 64, "vmcnt range");
};

template <int kX, int kMT, int kEpi>
__device__ __forceinline__ void dense_rows_body(const DenseArgs& g, lds_u8* lds) {
  using Cfg = CfgRows<kMT>;
  constexpr int kRN = Cfg::kRN;
  constexpr bool kGated = kEpi == kEpiGated;
  constexpr int R = Cfg::kRing, kTiles = kRN / 16;
  constexpr int kCols = kGated ? kRN / 2 : kRN;  // result columns
  const int lane = lane_id(), wave = wave_id();
  lds_u8* const own = lds + wave * Cfg::kWaveLds;
  const int n0 = blockIdx.x * kCols;
  // The slice's steps, of which this wave takes every fourth from its own on.
  const int all = (int)(((long long)g.K + 63) / 64);
  const int first = blockIdx.y * g.slice_steps;
  const int last = min(all, first + g.slice_steps);
  const int mine = max(0, (last - first - wave + 3) / 4);

  // DMA: an instruction has eight rows; lane l row l / 8, slot l % 8, which holds chunk
  // (l % 8) ^ slot_xor(row) (layout.hpp).
  const int drow = lane >> 3;
  const int chunk[2] = {(lane & 7) ^ slot_xor(drow), (lane & 7) ^ slot_xor(8 + drow)};
  const int rows = min(kCols, g.N - n0);
  const uint8_t* const w0 = g.b + (long long)n0 * g.ldb;
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(w0, (uint32_t)rows * (uint32_t)g.ldb);
  const __amdgpu_buffer_rsrc_t ru =
      kGated ? make_rsrc(w0 + g.up, (uint32_t)rows * (uint32_t)g.ldb) : rw;
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(g.a, (uint32_t)g.M * (uint32_t)g.lda);
  const int rot = (int)((blockIdx.x & 7u) * (unsigned)mine / 8u);
  auto fetch = [&](int s, int stage) {
    const int turned = s + rot < mine ? s + rot : s + rot - mine;
    const int k = (first + wave + 4 * turned) * 64;
    uint32_t oob[2];
#pragma unroll
    for (int p = 0; p < 2; ++p)
      oob[p] = s < mine && k + chunk[p] * 8 < g.K ? 0u : kOobOffset;
    const uint32_t so = s < mine ? (uint32_t)k * 2u : 0u;
    lds_u8* const to = own + stage * Cfg::kStage;
#pragma unroll
    for (int q = 0; q < kRN / 8; ++q) {
      const bool up = kGated && 8 * q >= kCols;
      const uint32_t v = (uint32_t)(8 * q - (up ? kCols : 0) + drow) * (uint32_t)g.ldb +
                         chunk[q & 1] * 16;
      dma16_nt(up ? ru : rw, to + q * 1024, v | oob[q & 1], so);
    }
#pragma unroll
    for (int q = 0; q < 2 * kMT; ++q) {
      const uint32_t v = (uint32_t)(8 * q + drow) * (uint32_t)g.lda + chunk[q & 1] * 16;
      dma16(rx, to + (kRN + 8 * q) * 128, v | oob[q & 1], so);
    }
  };

  const int r16 = lane & 15, grp = lane >> 4;
  f32x4 acc[kTiles][kMT] = {};
  auto compute = [&](int stage, int next) {
    const lds_u8* const from = own + stage * Cfg::kStage + r16 * 128;
    i32x4 fw[kTiles][2], fx[kMT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = ((2 * grp + h) ^ slot_xor(r16)) * 16;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) fw[t][h] = lds_read16(from + t * 2048 + at);
#pragma unroll
      for (int m = 0; m < kMT; ++m) fx[m][h] = lds_read16(from + (kTiles + m) * 2048 + at);
    }
    // The stage is free once the wave's reads are done.
    wait_lgkmcnt<0>();
    fetch(next, stage);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int m = 0; m < kMT; ++m)
          acc[t][m] = mfma_16x16x32<kX>(fw[t][h], fx[m][h], acc[t][m]);
  };
#pragma unroll
  for (int s = 0; s < R; ++s) fetch(s, s);
  for (int s = 0; s < mine; s += R) {
    static_for<R>([&](auto j) {
      if (s + j < mine) {
        wait_vmcnt<(R - 1) * Cfg::kDma>();
        compute(j, s + j + R);
      }
    });
  }
  // Everything fetched has landed, the empty steps' zeros too: the ring becomes the sums'
  // place, [wave][row of x][column].
  wait_vmcnt<0>();
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int m = 0; m < kMT; ++m)
      *reinterpret_cast<__attribute__((address_space(3))) f32x4*>(
          own + ((16 * m + r16) * kRN + 16 * t + 4 * grp) * 4) = acc[t][m];
  __syncthreads();
  const int count = g.M * kCols;
  for (int i = threadIdx.x; i < count; i += 64 * Cfg::kWaves) {
    const int row = i / kCols, c = i % kCols, col = n0 + c;
    if (col >= g.N) continue;
    float v = 0.0f, u = 0.0f;
#pragma unroll
    for (int w = 0; w < Cfg::kWaves; ++w) {
      const lds_u8* const p = lds + w * Cfg::kWaveLds + (row * kRN + c) * 4;
      v += __builtin_bit_cast(float, lds_read4(p));
      if constexpr (kGated) u += __builtin_bit_cast(float, lds_read4(p + kCols * 4));
    }
    if (gridDim.y > 1) {
      float* const to = g.partial + ((long long)blockIdx.y * g.M + row) * g.ldpart + col;
      to[0] = v;
      if constexpr (kGated) to[g.ldpart / 2] = u;
    } else {
      finish1<kEpi>(g.epi, dense_at(g.epi, row, col), 0, col, v, u);
    }
  }
}

}  // namespace detail
}  // namespace hipgemm
