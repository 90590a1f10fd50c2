// Streams quantised weights past a few rows of 16-bit activations: the inner
// part of the products with 4-bit weights for 5 rows and more, and of the
// experts' products.
//
// What bounds it is the weights' bytes, 9 per CU and cycle at most, so all that
// matters is that enough of them are on their way all the time, from the first
// instruction to the last.  One workgroup per CU works off a list of items (32
// kWN rows of weights times a group of rows of x); each wave reads its own
// weights straight into registers, kRing units ahead, across the items' ends, and
// has no other loads of memory in between.  Activations lie in LDS, all of the
// item's K, and stay there for all items of a group.
//
// A wave multiplies kMT tiles of 16 rows of x by 2 tiles of 16 rows of weights,
// v_mfma_f32_16x16x32.  kWK waves take turns over K, and their sums meet in LDS at
// an item's end; kWN sets of them have rows of weights of their own.  K goes in
// units of two blocks of 128: lane (r, g) = (l % 16, l / 16) reads the 32 weights
// k = 32 g .. + 31 of row r of a tile and block, 16 bytes (32 for e4m3), so that a
// wave takes whole 128-byte lines of rows, and the four MFMAs of a block take 8 of
// each lane's 32 (any order of K will do, as long as the activations are read in
// the same).
//
// Scales are applied in fp32 to the sum over one group.  A lane loads the scale
// (and zero point) of its 32 weights, one load per tile and block, and there are
// four ways on from there, by what a block's groups are:
//   kNone    e4m3: scales belong to whole rows, applied at the end.
//   kCoarse  groups of a multiple of 128: the four lane groups' scales are the
//            same, applied to the four MFMAs' sum.
//   kFine    any multiple of 32: each MFMA's sum is scaled by itself, so it has
//            to hold 32 neighbouring k.  The codes get there by a transpose of
//            4 x 4 dwords over the four lane groups, four swaps in all
//            (v_permlane32_swap, v_permlane16_swap), the scales by three.
//   kInline  fp4 with E8M0 scales and bf16 activations: the conversion
//            multiplies by the scale, exactly, as a power of two and a 2-bit
//            significand are a bf16 number wherever the product is one.
// The int4 excess (decode.hpp) needs the group's sum of x per row: one more
// MFMA by ones gives it in the accumulators' own layout.
#pragma once

#include "decode.hpp"

namespace hipgemm {
namespace detail {

constexpr int kNone = 0, kCoarse = 1, kFine = 2, kInline = 3;

// v[j] of lane group g <- v[g] of lane group j.
__device__ __forceinline__ void transpose4(uint32_t (&v)[4]) {
  const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  v[0] = c[0];
  v[1] = c[1];
  v[2] = d[0];
  v[3] = d[1];
}
// to[g] = lane group g's v, in all lane groups.
__device__ __forceinline__ void spread4(uint32_t v, uint32_t (&to)[4]) {
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const auto b = __builtin_amdgcn_permlane16_swap(a[0], a[0], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[1], a[1], false, false);
  to[0] = b[0];
  to[1] = b[1];
  to[2] = c[0];
  to[3] = c[1];
}

template <int kS>
__device__ __forceinline__ uint32_t scale_raw(const uint8_t* p, int i) {
  if constexpr (type_bytes(kS) == 4) return reinterpret_cast<const uint32_t*>(p)[i];
  else if constexpr (type_bytes(kS) == 2) return reinterpret_cast<const uint16_t*>(p)[i];
  else return p[i];
}
// kLo: activations in two parts, x = hi + lo (16 bits each).
// kWaves = kWK kWN waves.
template <int kX, int kW, int kS, int kMode, int kMT, bool kLo, int kWaves>
struct Stream {
  static constexpr int kWK = 8, kWN = kWaves / kWK, kNT = 2;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kWords = kW == kWE4M3 ? 2 : 1;  // 16-byte loads of a lane's weights
  static constexpr int kParts = kLo ? 2 : 1;
  static constexpr int kRows = 16 * kMT;
  static constexpr int kTile = 32 * kWN;  // rows of weights of an item
  static constexpr int kRing = 2;         // units in flight per wave, of 4 or 8 KiB
  // LDS: activations (rows x parts of K, each row 16 bytes longer, so that the 16
  // rows' pieces of an MFMA operand lie on all banks) and the waves' sums.
  static constexpr int kSumBytes = kWaves * kNT * kMT * kWave * 16;
  static constexpr int kPadBytes = kRows * kParts * 16;
  // Of 160 KiB, 8 for the kernel's own tables; at most 16 rows of 4096.
  static constexpr int kRoom = (152 << 10) - kSumBytes - kPadBytes;
  static constexpr int kElems = (kRoom > 2 << 16 ? 2 << 16 : kRoom) / 512 * 256;
  static constexpr int kXBytes = 2 * kElems + kPadBytes;
  static constexpr int kLdsBytes = kXBytes + kSumBytes;
  // Rows of a group whose K elements fit.
  __host__ __device__ static int rows_that_fit(int k_len) {
    const int r = kElems / (kParts * ((k_len + 255) & ~255));
    return r < kRows ? r : kRows;
  }

  // Set by the kernel.
  lds_u8* lds;
  int K;
  float inv;  // 32 / group

  // This lane's rows of weights, scales and zero points, of the item being
  // loaded: row l % 16 of each tile.
  const uint8_t* w[kNT];
  const uint8_t* s[kNT];
  const uint8_t* z[kNT];
  f32x4 acc[kNT][kMT];

  struct Unit {
    i32x4 w[kNT][2][kWords];
    uint32_t s[kNT][2], z[kNT][2];
  };

  // kb: first k of the unit, a multiple of 256.  Past k_end its last 32 are read
  // again.
  __device__ __forceinline__ void load(Unit& b, int kb, int k_end) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = min(kb + 128 * h + 32 * (lane_id() >> 4), k_end - 32);
      const int grp = kMode == kNone ? 0 : group_of(k >> 5, inv);
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const uint8_t* p = w[n] + (kW == kWE4M3 ? k : k >> 1);
#pragma unroll
        for (int i = 0; i < kWords; ++i)
          b.w[n][h][i] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(p) + i);
        if (kMode != kNone || h == 0) b.s[n][h] = scale_raw<kS>(s[n], grp);
        if constexpr (kW == kWInt4Z) b.z[n][h] = z[n][grp];
      }
    }
  }

  // k0 to below k1 of `rows` rows of x to LDS, zeros from there to the next
  // multiple of 256.  row_at(part, row): the row's address, the same for the whole
  // wave.
  __device__ __forceinline__ int pitch(int len) const { return 2 * ((len + 255) & ~255) + 16; }
  template <class F>
  __device__ __forceinline__ void fetch_x(int k0, int k1, int rows, F&& row_at) const {
    const int wave = wave_id(), kl = 8 * lane_id();
    const int segs = (k1 - k0 + 511) >> 9, units = segs * rows * kParts, pt = pitch(k1 - k0);
    constexpr int kAhead = 7;  // 16 waves: all of LDS in one go
    for (int u = wave; u < units; u += kAhead * kWaves) {
      i32x4 v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int t = min(u + i * kWaves, units - 1), row = t / segs;
        const uint8_t* p = row_at(row / rows, row % rows);
        v[i] = *reinterpret_cast<const i32x4*>(p + 2ll * min(k0 + (t - row * segs) * 512 + kl, K - 8));
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int t = min(u + i * kWaves, units - 1), row = t / segs;
        const int k = (t - row * segs) * 512 + kl;
        if (k < ((k1 - k0 + 255) & ~255))
          *reinterpret_cast<__attribute__((address_space(3))) i32x4*>(lds + row * pt + 2 * k) =
              k0 + k < k1 ? pair_order<kW>(v[i]) : i32x4{};
      }
    }
  }

  // Block h of a unit, at kb; from: this lane's row of x at it.
  __device__ __forceinline__ void mul(const Unit& b, int h, int kb, const lds_u8* from,
                                      int part_bytes, const int (&tile)[kMT]) {
    const int g = lane_id() >> 4;
    uint32_t q[kNT][4 * kWords];
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4 * kWords; ++i) q[n][i] = (uint32_t)b.w[n][h][i / 4][i % 4];
    if constexpr (kW == kWE4M3) {
      if (kb + 128 > K && kb + 32 * g >= K) {  // a NaN code times zero would stay one
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int i = 0; i < 8; ++i) q[n][i] = 0u;
      }
    }
    uint32_t sc[kNT][4], zp[kNT][4];
    if constexpr (kMode == kFine) {
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        uint32_t t[4] = {q[n][0], q[n][1], q[n][2], q[n][3]};
        transpose4(t);
#pragma unroll
        for (int i = 0; i < 4; ++i) q[n][i] = t[i];
        spread4(b.s[n][h], sc[n]);
        if constexpr (kW == kWInt4Z) spread4(b.z[n][h], zp[n]);
      }
    }
    // Sums of the block's group: the accumulators themselves where no scale is
    // to be applied here.
    f32x4 part[kNT][kMT], xs[kMT];
    const lds_u8* at = from + (kMode == kFine ? 16 * g : 64 * g);
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
        for (int m = 0; m < kMT; ++m)
          a[p][m] = lds_read16(at + p * part_bytes + tile[m] + (kMode == kFine ? 64 * j : 16 * j));
      if constexpr (is_int4(kW)) {
        const int one = (int)kOnes2<kX>;
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
          for (int m = 0; m < kMT; ++m)
            xs[m] = mfma_16x16x32<kX>(a[p][m], i32x4{one, one, one, one}, xs[m]);
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const float c = kMode == kInline ? scale_of<kS>(b.s[n][h]) : 1.0f;
        const i32x4 v = kW == kWE4M3 ? decode8<kX, kW>(q[n][kWords * j], q[n][kWords * j + kWords - 1], c)
                                     : decode8<kX, kW>(q[n][j], 0u, c);
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
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            const float c = scale_of<kS>(kMode == kFine ? sc[n][j] : b.s[n][h]);
            float off = -(kInt4Bias<kX> + 8.0f);
            if constexpr (kW == kWInt4Z)
              off = -(kInt4Bias<kX> + (float)(kMode == kFine ? zp[n][j] : b.z[n][h]));
#pragma unroll
            for (int m = 0; m < kMT; ++m)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float t = part[n][m][e];
                if constexpr (is_int4(kW)) t = __builtin_fmaf(off, xs[m][e], t);
                acc[n][m][e] = __builtin_fmaf(c, t, acc[n][m][e]);
              }
          }
        }
      }
    }
  }

  // Items first to below last, each over len (a multiple of 256, or up to K) of K.
  // p.weights(item): sets w, s, z;  p.k_begin(item): its first k;
  // p.group(item): of items that share x;  p.rows(group), p.row_at(group, part, row);
  // p.finish(item): the item's sums are in LDS (sum_of).
  template <class P>
  __device__ __forceinline__ void run(int first, int last, int len, P& p) {
    if (first >= last) return;
    const int wave = wave_id(), wk = wave % kWK;
    const int turns = (((len + 255) >> 8) + kWK - 1) / kWK;  // a wave's units of an item
    int li = first, lu = 0, lk = 0, lend = 0;  // the item and unit that is loaded next
    auto next_item = [&]() {
      // (past the last item: a place that was read before)
      if (li < last) {
        p.weights(li);
        lk = p.k_begin(li);
        lend = min(lk + len, K);
        lk += wk * 256;
      } else {
        lend = 32;
      }
    };
    next_item();
    Unit ring[kRing];
    auto fetch = [&](Unit& b) {
      load(b, lk + lu * kWK * 256, lend);
      if (++lu == turns) {
        lu = 0;
        ++li;
        next_item();
      }
    };
#pragma unroll
    for (int i = 0; i < kRing; ++i) fetch(ring[i]);

    int item = first, u = 0, group = -1, part_bytes = 0, k0 = 0, k1 = 0;
    int tile[kMT];
    const lds_u8* row = lds;
    for (;;) {
#pragma unroll
      for (int r = 0; r < kRing; ++r) {
        if (u == 0) {
          k0 = p.k_begin(item);
          k1 = min(k0 + len, K);
          if (p.group(item) != group) {
            group = p.group(item);
            const int rows = p.rows(group);
            barrier();  // the group before has been read
            fetch_x(k0, k1, rows, [&](int part, int m) { return p.row_at(group, part, m); });
            wait_lgkmcnt<0>();
            barrier();
            // (rows that are not there: the last one again)
            const int pt = pitch(k1 - k0), lr = min(lane_id() & 15, rows - 1);
            part_bytes = rows * pt;
            row = lds + lr * pt;
#pragma unroll
            for (int m = 0; m < kMT; ++m)
              tile[m] = (min(16 * m + (lane_id() & 15), rows - 1) - lr) * pt;
          }
#pragma unroll
          for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int m = 0; m < kMT; ++m) acc[n][m] = f32x4{};
        }
        Unit& b = ring[r];
        const int kb = k0 + (u * kWK + wk) * 256;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (kb + 128 * h < k1) mul(b, h, kb + 128 * h, row + 2 * (kb + 128 * h - k0), part_bytes, tile);
        const bool end = ++u == turns;
        if constexpr (kMode == kNone) {
          if (end) {
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
              for (int m = 0; m < kMT; ++m) acc[n][m] *= scale_of<kS>(b.s[n][0]);
          }
        }
        fetch(b);
        if (end) {
          spill_sums(wave);
          p.finish(item);
          u = 0;
          if (++item == last) return;
        }
      }
    }
  }

  // The waves' accumulators to LDS: [wave][n][m][row][column], 16 x 16 floats a
  // tile (wave = wn kWK + wk).
  __device__ __forceinline__ void spill_sums(int wave) const {
    barrier();  // the item before has been finished
    const int r = lane_id() & 15, g = lane_id() >> 4;
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int m = 0; m < kMT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<__attribute__((address_space(3))) float*>(
              lds + kXBytes + ((((wave * kNT + n) * kMT + m) * 16 + 4 * g + e) * 16 + r) * 4) =
              acc[n][m][e];
    wait_lgkmcnt<0>();
    barrier();
  }
  // The sum over K of tile n of set wn.
  __device__ __forceinline__ float sum_of(int wn, int n, int m, int row, int col) const {
    float v = 0.0f;
#pragma unroll
    for (int q = 0; q < kWK; ++q)
      v += *reinterpret_cast<const __attribute__((address_space(3))) float*>(
          lds + kXBytes + (((((wn * kWK + q) * kNT + n) * kMT + m) * 16 + row) * 16 + col) * 4);
    return v;
  }
};

}  // namespace detail
}  // namespace hipgemm
