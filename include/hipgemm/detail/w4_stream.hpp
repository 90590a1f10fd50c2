// Streams quantised weights past a few rows of 16-bit activations: the inner
// part of the products with 4-bit weights for 5 rows and more, and of the
// experts' products.
//
// A wave multiplies kMT tiles of 16 rows of x by kNT tiles of 16 rows of
// weights, v_mfma_f32_16x16x32, straight from memory to registers: nothing is
// shared between waves but activations, which come from the L1 and L2.  K goes
// in blocks of 128: lane (r, g) = (l % 16, l / 16) reads the 32 weights k = 32 g
// .. + 31 of row r of a tile, 16 bytes (32 for e4m3), so that a wave takes whole
// 64-byte pieces of rows, and the four MFMAs of a block take 8 of each lane's
// 32 (any order of K will do, as long as the activations are read in the same).
// The next blocks' loads are in flight while a block is multiplied.
//
// Scales are applied in fp32 to the sum over one group, and there are three
// ways, by what a block's groups are:
//   kNone    e4m3: scales belong to whole rows (left to the caller).
//   kCoarse  groups of a multiple of 128: one scale per row of weights and
//            block, on the four MFMAs' sum.
//   kFine    any multiple of 32: each MFMA's sum is scaled by itself, so it has
//            to hold 32 neighbouring k.  The codes get there by a transpose of
//            4 x 4 dwords over the four lane groups, four swaps in all
//            (v_permlane32_swap, v_permlane16_swap).
//   kInline  fp4 with E8M0 scales and bf16 activations: the conversion
//            multiplies by the scale, exactly, as a power of two and a 2-bit
//            significand are a bf16 number wherever the product is one (a group
//            is a lane's 32 or more).
// The int4 excess (decode.hpp) needs the group's sum of x per row: one more
// MFMA by ones gives it in the accumulators' own layout.
#pragma once

#include "decode.hpp"

namespace hipgemm {
namespace detail {

constexpr int kNone = 0, kCoarse = 1, kFine = 2, kInline = 3;

// v[j] of lane group g <- v[g] of lane group j.
__device__ __forceinline__ void transpose4(uint32_t (&v)[4]) {
  auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
  auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  v[0] = c[0];
  v[1] = c[1];
  v[2] = d[0];
  v[3] = d[1];
}

template <int kS>
__device__ __forceinline__ uint32_t scale_raw(const uint8_t* p, int i) {
  if constexpr (type_bytes(kS) == 4) return reinterpret_cast<const uint32_t*>(p)[i];
  else if constexpr (type_bytes(kS) == 2) return reinterpret_cast<const uint16_t*>(p)[i];
  else return p[i];
}
template <int kS>
__device__ __forceinline__ float scale_of(uint32_t r) {
  if constexpr (kS == kInF32) return __builtin_bit_cast(float, r);
  else if constexpr (kS == kInBf16) return __builtin_bit_cast(float, r << 16);
  else if constexpr (kS == kInF16) return (float)__builtin_bit_cast(_Float16, (uint16_t)r);
  else
    return __builtin_bit_cast(float, r == 255u ? 0x7fc00000u : r == 0u ? 0x00400000u : r << 23);
}

// The scale group of unit u of 32 weights, inv = 1 / (units per group): exact
// for u < 2^21 (the quotient is 0.5 / group or more from an integer, its error
// below u / group 2^-22).
__device__ __forceinline__ int group_of(int u, float inv) {
  return (int)(((float)u + 0.5f) * inv);
}

// kLo: activations in two parts, x = hi + lo (16 bits each, at x and x + lo).
template <int kX, int kW, int kS, int kMode, int kNT, int kMT, bool kLo>
struct Stream {
  static constexpr int kWords = kW == kWE4M3 ? 2 : 1;  // 16-byte loads of a lane's weights
  static constexpr int kParts = kLo ? 2 : 1;
  static constexpr int kSc = kMode == kNone ? 0 : kMode == kFine ? 4 : 1;

  // This lane's rows: weights, scales and zero points of row l % 16 of each
  // weight tile, activations of row l % 16 of each tile of x.
  const uint8_t* w[kNT];
  const uint8_t* s[kNT];
  const uint8_t* z[kNT];  // null: 8
  const uint8_t* x[kMT];
  long long lo;  // bytes from an activation's high part to its low part
  int K;
  float inv;     // 32 / group
  f32x4 acc[kNT][kMT] = {};

  struct Block {
    i32x4 w[kNT][kWords];
    i32x4 x[kParts][kMT][4];
    uint32_t s[kNT][kSc ? kSc : 1];
    uint32_t z[kNT][kSc ? kSc : 1];
  };

  // kb: first k of the block, a multiple of 128; beyond K nothing is read that
  // is not (the last 32 of K are read again, and masked in mul).
  __device__ __forceinline__ void load(Block& b, int kb) const {
    const int g = lane_id() >> 4;
    const int k = min(kb + 32 * g, K - 32);
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const uint8_t* p = w[n] + (kW == kWE4M3 ? k : k >> 1);
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        b.w[n][i] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(p) + i);
    }
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
      for (int m = 0; m < kMT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint8_t* a = x[m] + p * lo;
          if constexpr (kMode == kFine)
            b.x[p][m][j] = *reinterpret_cast<const i32x4*>(a + 2 * (min(kb + 32 * j, K - 32) + 8 * g));
          else
            b.x[p][m][j] = *reinterpret_cast<const i32x4*>(a + 2 * k + 16 * j);
        }
    if constexpr (kMode != kNone) {
#pragma unroll
      for (int j = 0; j < kSc; ++j) {
        const int at = kMode == kInline ? k : min(kb + 32 * j, K - 32);
        const int grp = group_of(at >> 5, inv);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          b.s[n][j] = scale_raw<kS>(s[n], grp);
          if constexpr (kW == kWInt4) b.z[n][j] = z[n] ? (uint32_t)z[n][grp] : 8u;
        }
      }
    }
  }

  __device__ __forceinline__ void mul(Block& b, int kb) {
    if (kb + 128 > K) {  // the last block of a K that is no multiple of 128
      const int g = lane_id() >> 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = kMode == kFine ? kb + 32 * j < K : kb + 32 * g < K;
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
          for (int m = 0; m < kMT; ++m) b.x[p][m][j] = in ? b.x[p][m][j] : i32x4{};
      }
      if constexpr (kW == kWE4M3) {  // a NaN code times zero would stay one
        const bool in = kb + 32 * g < K;
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int i = 0; i < kWords; ++i) b.w[n][i] = in ? b.w[n][i] : i32x4{};
      }
    }
    uint32_t q[kNT][8];
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4 * kWords; ++i) q[n][i] = (uint32_t)b.w[n][i / 4][i % 4];
    if constexpr (kMode == kFine)
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        uint32_t t[4] = {q[n][0], q[n][1], q[n][2], q[n][3]};
        transpose4(t);
#pragma unroll
        for (int i = 0; i < 4; ++i) q[n][i] = t[i];
      }
    // Sums of the block's group: the accumulators themselves where no scale is
    // to be applied here.
    f32x4 part[kNT][kMT], xs[kMT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (kMode == kFine || j == 0) {
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          xs[m] = f32x4{};
#pragma unroll
          for (int n = 0; n < kNT; ++n) part[n][m] = f32x4{};
        }
      }
      i32x4 a[kParts][kMT];
#pragma unroll
      for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int m = 0; m < kMT; ++m) a[p][m] = pair_order<kW>(b.x[p][m][j]);
      if constexpr (kW == kWInt4) {
        const int one = (int)kOnes2<kX>;
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
          for (int m = 0; m < kMT; ++m)
            xs[m] = mfma_16x16x32<kX>(a[p][m], i32x4{one, one, one, one}, xs[m]);
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const float sc = kMode == kInline ? scale_of<kS>(b.s[n][0]) : 1.0f;
        const i32x4 v = kW == kWE4M3 ? decode8<kX, kW>(q[n][2 * j], q[n][2 * j + 1], sc)
                                     : decode8<kX, kW>(q[n][j], 0u, sc);
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
          for (int m = 0; m < kMT; ++m) {
            if constexpr (kMode == kNone || kMode == kInline)
              acc[n][m] = mfma_16x16x32<kX>(a[p][m], v, acc[n][m]);
            else
              part[n][m] = mfma_16x16x32<kX>(a[p][m], v, part[n][m]);
          }
      }
      if constexpr (kMode == kFine || kMode == kCoarse) {
        if (kMode == kFine || j == 3) {
          const int c = kMode == kFine ? j : 0;
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            const float sc = scale_of<kS>(b.s[n][c]);
            const float off = -(kInt4Bias<kX> + (float)(kW == kWInt4 ? b.z[n][c] : 0u));
#pragma unroll
            for (int m = 0; m < kMT; ++m)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float t = part[n][m][e];
                if constexpr (kW == kWInt4) t = __builtin_fmaf(off, xs[m][e], t);
                acc[n][m][e] = __builtin_fmaf(sc, t, acc[n][m][e]);
              }
          }
        }
      }
    }
  }

  // Pairs of blocks first, first + step, ... below end (a pair is 256 of K: the
  // halves of 4-bit weights' 128-byte lines).
  __device__ __forceinline__ void run(int first, int end, int step) {
    if (first >= end) return;
    Block b[2], c[2];
    load(b[0], first * 256);
    load(b[1], first * 256 + 128);
    for (int pair = first; pair < end; pair += step) {
      // (past the end: the last weights again, not used)
      const int next = min(pair + step, end - 1);
      load(c[0], next * 256);
      load(c[1], next * 256 + 128);
      mul(b[0], pair * 256);
      if (pair * 256 + 128 < K) mul(b[1], pair * 256 + 128);
      b[0] = c[0];
      b[1] = c[1];
    }
  }
  __device__ __forceinline__ int pairs() const { return (K + 255) >> 8; }
};

}  // namespace detail
}  // namespace hipgemm
