// Streams quantised weights past a few rows of 16-bit activations: the inner
// part of the experts' products where they are grouped (moe.hpp).
//
// What bounds it is the weights' bytes, 9 per CU and cycle at most, so all that
// matters is that enough of them are on their way all the time, from the first
// instruction to the last.  One workgroup per CU works off a list of items (32
// kWN rows of weights times a group of rows of x); kWK of its eight waves take
// turns over K, and their sums meet in LDS at an item's end, kWN = 8 / kWK sets of
// them have 32 rows of weights of their own.  Each wave brings its own weights
// into its own ring of LDS by DMA, two units of 4 KiB ahead, across the items'
// ends, and has hardly any other loads of memory in between.  Activations lie in
// LDS, all of the item's K, and stay there for all items of a group.
//
// A unit is 32 rows by 128 bytes: whole lines, eight lanes to each, which reach
// 6.0 TB/s from memory where an MFMA operand's own order (16 rows, 64 bytes of
// each) stops at 5.1; non-temporal loads, plain ones reach half (64 MiB, one load
// of 16 KiB per wave, all at once).  A wave multiplies kMT tiles of 16 rows of x
// by the unit's two tiles of 16 rows, v_mfma_f32_16x16x32: lane (r, g) = (l % 16,
// l / 16) takes 32 weights of a row (16 bytes at chunk 4 h + g of the line in block
// h; for e4m3 the chunks g and g + 4, one block), and the four MFMAs of a block
// take 8 of each lane's 32 (any order of K will do, as long as the activations
// are read in the same).  A line's chunk c lies at slot c ^ (row % 8), which makes
// these reads free of bank conflicts.
//
// Scales are applied in fp32 to the sum over one group, in four ways, by what a
// block's groups are:
//   kNone    e4m3: scales belong to whole rows, applied at the end.
//   kCoarse  groups of a multiple of 128: one scale per row and block, on the four
//            MFMAs' sum.  One load brings those of a unit (two tiles, two blocks:
//            one each per lane group), three swaps spread them.
//   kFine    any multiple of 32: each MFMA's sum is scaled by itself, so it has
//            to hold 32 neighbouring k.  The codes get there by a transpose of
//            4 x 4 dwords over the four lane groups, four swaps in all
//            (v_permlane32_swap, v_permlane16_swap), the scales by three.
//            A load per tile and block, a lane the scale of its 32 weights.
//   kInline  fp4 with E8M0 scales and bf16 activations: the conversion
//            multiplies by the scale, exactly, as a power of two and a 2-bit
//            significand are a bf16 number wherever the product is one.  Loads as
//            for kFine.
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
// kParts: activations in that many parts, x their sum (16 bits each).
// kTables: bytes of LDS that the kernel keeps for itself.
template <int kX, int kW, int kS, int kMode, int kMT, int kParts, int kWK, int kTables>
struct Stream {
  static constexpr int kWaves = 8, kThreads = kWaves * kWave, kNT = 2;
  static constexpr int kRows = 16 * kMT;
  static constexpr int kWN = kWaves / kWK;
  static constexpr int kTile = 32 * kWN;  // rows of weights of an item
  static constexpr int kBlocks = kW == kWE4M3 ? 1 : 2;  // of 128 of K, of a unit
  static constexpr int kUnit = 128 * kBlocks;
  static constexpr int kUnitBytes = 4096;
  static constexpr int kRing = 2;
  // LDS: activations (rows x parts of K, each row 16 bytes longer, so that the 16
  // rows' pieces of an MFMA operand lie on all banks), rings, the waves' sums, the
  // kernel's tables: 160 KiB in all.
  static constexpr int kRingBytes = kWaves * kRing * kUnitBytes;
  static constexpr int kSumBytes = kWaves * kNT * kMT * kWave * 16;
  static constexpr int kPadBytes = kRows * kParts * 16;
  static constexpr int kElems = ((160 << 10) - kTables - kRingBytes - kSumBytes - kPadBytes) / 512 * 256;
  static constexpr int kXBytes = 2 * kElems + kPadBytes;
  static constexpr int kSums = kSumBytes / 4;
  // Rows of a group whose K elements fit.
  __host__ __device__ static int rows_that_fit(int k_len) {
    const int r = kElems / (kParts * ((k_len + 255) & ~255));
    return r < kRows ? r : kRows;
  }
  // Loads of scales and zero points of a unit.
  static constexpr int kSc = kMode == kFine || kMode == kInline ? 4 : 1;

  // Set by the kernel: three objects of LDS of its own (the compiler waits for
  // DMAs before it stores to the object that they fill).
  lds_u8* lds;        // kXBytes
  lds_u8* rings;      // kRingBytes
  __attribute__((address_space(3))) float* sums;  // kSums
  int K;
  float inv;     // 32 / group
  uint32_t ldw;  // bytes of a row of weights

  // The item being loaded: its two tiles' rows, and this lane's rows of scales and
  // zero points (set_rows).
  __amdgpu_buffer_rsrc_t wb[kNT];
  const uint8_t* sp[kNT];
  const uint8_t* zp[kNT];
  f32x4 acc[kNT][kMT];

  struct Scales {
    uint32_t s[kSc], z[kSc];
  };

  // This wave's set of rows.
  __device__ static int set() { return wave_id() / kWK; }
  // The tile of this lane's scales: one load each for both tiles, or one in all.
  __device__ static int scale_tile(int n) {
    const int g = lane_id() >> 4;
    return kMode == kCoarse ? g >> 1 : kMode == kNone ? g & 1 : n;
  }
  // Tile n: 16 rows at w.
  __device__ __forceinline__ void set_tile(int n, const uint8_t* w) {
    wb[n] = make_rsrc(w, 16 * ldw);
  }

  // The unit at k to the ring's slot; past k_end nothing is fetched.  Always
  // kLoads loads, in this order: the wait for a unit counts those of the next.
  static constexpr int kLoads = 4 + kSc * (kW == kWInt4Z ? 2 : 1);
  __device__ __forceinline__ void load(Scales& b, lds_u8* slot, int k, int k_end) const {
    const int lane = lane_id(), g = lane >> 4;
    const int row = lane >> 3, chunk = (lane & 7) ^ row;
    const int kc = k + chunk * (kW == kWE4M3 ? 16 : 32);
    const uint32_t vo = kc < k_end ? (uint32_t)row * ldw + (kW == kWE4M3 ? kc : kc >> 1) : kOobOffset;
    compiler_fence();
    sched_fence();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      dma16_nt(wb[i >> 1], slot + 1024 * i, vo, (i & 1) * 8 * ldw);
    compiler_fence();
    sched_fence();
#pragma unroll
    for (int i = 0; i < kSc; ++i) {
      // (clamped: past the end the last scales once more)
      const int h = kMode == kCoarse ? g & 1 : i & 1;
      const int at = kMode == kCoarse ? k + 128 * h : k + 128 * h + 32 * g;
      const int grp = kMode == kNone ? 0 : group_of(max(min(at, k_end - 32), 0) >> 5, inv);
      b.s[i] = scale_raw<kS>(sp[kSc == 4 ? i >> 1 : 0], grp);
      if constexpr (kW == kWInt4Z) b.z[i] = zp[kSc == 4 ? i >> 1 : 0][grp];
    }
    compiler_fence();
    sched_fence();
  }

  // k0 to below k1 of `rows` rows of x to LDS, zeros from there to the next
  // multiple of 256.  row_at(part, row): the row's address, the same for the whole
  // wave.
  __device__ __forceinline__ int pitch(int len) const { return 2 * ((len + 255) & ~255) + 16; }
  template <class F>
  __device__ __forceinline__ void fetch_x(int k0, int k1, int rows, F&& row_at) const {
    const int wave = wave_id(), kl = 8 * lane_id();
    const int segs = (k1 - k0 + 511) >> 9, units = segs * rows * kParts, pt = pitch(k1 - k0);
    constexpr int kAhead = 8;
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
              k0 + k < k1 ? v[i] : i32x4{};
      }
    }
  }

  // Reads of LDS in the loop, in assembly with their wait: before a read that the
  // compiler knows of it waits for all DMAs into LDS, those of the unit behind
  // among them.  read_lines: 16 bytes each of rows r and 16 + r of a unit;  read_x:
  // the four MFMAs' operands of a row of x.
  __device__ static void read_x(const lds_u8* p, i32x4 (&v)[4]) {
    if constexpr (kW == kWE4M3)
      asm volatile(
          "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:16\n\t"
          "ds_read_b128 %2, %4 offset:128\n\tds_read_b128 %3, %4 offset:144\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
          : "v"(p)
          : "memory");
    else if constexpr (kMode == kFine)
      asm volatile(
          "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:64\n\t"
          "ds_read_b128 %2, %4 offset:128\n\tds_read_b128 %3, %4 offset:192\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
          : "v"(p)
          : "memory");
    else
      asm volatile(
          "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:16\n\t"
          "ds_read_b128 %2, %4 offset:32\n\tds_read_b128 %3, %4 offset:48\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
          : "v"(p)
          : "memory");
  }
  __device__ static void read_lines(const lds_u8* p, i32x4 (&v)[kNT]) {
    asm volatile(
        "ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:2048\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(v[0]), "=&v"(v[1])
        : "v"(p)
        : "memory");
  }

  // Block h of the unit in slot, scales sc and zero points zp (by tile and block,
  // or for kFine by tile and MFMA, in all lanes of a row); from: this lane's row of
  // x at the block.
  __device__ __forceinline__ void mul(const lds_u8* slot, int h, const uint32_t (&sc)[kNT][4],
                                      const uint32_t (&zs)[kNT][4], const lds_u8* from,
                                      int part_bytes, const int (&tile)[kMT]) {
    const int r = lane_id() & 15, g = lane_id() >> 4;
    const lds_u8* line = slot + r * 128;
    i32x4 wa[kNT], wx[kNT];
    read_lines(line + 16 * ((4 * h + g) ^ (r & 7)), wa);
    if constexpr (kW == kWE4M3) read_lines(line + 16 * ((4 + g) ^ (r & 7)), wx);
    uint32_t q[kNT][8];
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q[n][i] = (uint32_t)wa[n][i];
        if constexpr (kW == kWE4M3) q[n][4 + i] = (uint32_t)wx[n][i];
      }
      if constexpr (kMode == kFine) {
        uint32_t t[4] = {q[n][0], q[n][1], q[n][2], q[n][3]};
        transpose4(t);
#pragma unroll
        for (int i = 0; i < 4; ++i) q[n][i] = t[i];
      }
    }
    // Sums of the block's group: the accumulators themselves where no scale is
    // to be applied here.
    f32x4 part[kNT][kMT], xs[kMT];
    const lds_u8* at = from + (kW == kWE4M3 ? 32 * g : kMode == kFine ? 16 * g : 64 * g);
    i32x4 a[kParts][kMT][4];
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
      for (int m = 0; m < kMT; ++m) read_x(at + p * part_bytes + tile[m], a[p][m]);
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
      if constexpr (is_int4(kW)) {
        const int one = (int)kOnes2<kX>;
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
          for (int m = 0; m < kMT; ++m)
            xs[m] = mfma_16x16x32<kX>(a[p][m][j], i32x4{one, one, one, one}, xs[m]);
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const float c = kMode == kInline ? scale_of<kS>(sc[n][h]) : 1.0f;
        const i32x4 v = kW == kWE4M3 ? decode8<kX, kW>(q[n][2 * j], q[n][2 * j + 1], c)
                                     : decode8<kX, kW>(q[n][j], 0u, c);
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
          for (int m = 0; m < kMT; ++m) {
            if constexpr (kMode == kNone || kMode == kInline)
              acc[n][m] = mfma_16x16x32<kX>(a[p][m][j], v, acc[n][m]);
            else
              part[n][m] = mfma_16x16x32<kX>(a[p][m][j], v, part[n][m]);
          }
      }
      if constexpr (kMode == kFine || kMode == kCoarse) {
        if (kMode == kFine || j == 3) {
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            const int i = kMode == kFine ? j : h;
            const float c = scale_of<kS>(sc[n][i]);
            float off = -8.0f;
            if constexpr (kW == kWInt4Z) off = -(float)zs[n][i];
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

  // A unit's scales by tile and block (kCoarse, kInline) or, for block h, by tile
  // and MFMA (kFine).
  __device__ __forceinline__ void spread(const uint32_t (&v)[kSc], int h, uint32_t (&to)[kNT][4]) const {
    if constexpr (kMode == kCoarse) {
      uint32_t t[4];
      spread4(v[0], t);
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        to[n][0] = t[2 * n];
        to[n][1] = t[2 * n + 1];
      }
    } else if constexpr (kMode == kInline) {
#pragma unroll
      for (int n = 0; n < kNT; ++n) to[n][h] = v[2 * n + h];
    } else if constexpr (kMode == kFine) {
#pragma unroll
      for (int n = 0; n < kNT; ++n) spread4(v[2 * n + h], to[n]);
    }
  }

  // Items first to below last, each over len (a multiple of 256, or up to K) of K.
  // p.weights(item): set_tile and the rows of scales;  p.k_begin(item): its first k;
  // p.group(item): of items that share x;  p.rows(group), p.row_at(group, part, row);
  // p.finish(item): the item's sums are in LDS (sum_of).
  template <class P>
  __device__ __forceinline__ void run(int first, int last, int len, P& p) {
    if (first >= last) return;
    const int wave = wave_id(), wk = wave % kWK;
    lds_u8* ring = rings + wave * kRing * kUnitBytes;
    const int turns = ((len + kUnit - 1) / kUnit + kWK - 1) / kWK;  // a wave's units of an item
    int li = first, lu = 0, lk = 0, lend = 0;  // the item and unit that is loaded next
    auto next_item = [&]() {
      if (li < last) {
        p.weights(li);
        lk = p.k_begin(li);
        lend = min(lk + len, K);
        lk += wk * kUnit;
      } else {
        lend = 0;
      }
    };
    next_item();
    auto fetch = [&](Scales& b, int slot) {
      load(b, ring + slot * kUnitBytes, lk + lu * kWK * kUnit, lend);
      if (++lu == turns) {
        lu = 0;
        ++li;
        next_item();
      }
    };
    Scales scales[kRing];
#pragma unroll
    for (int i = 0; i < kRing; ++i) fetch(scales[i], i);

    int item = first, u = 0, group = -1, part_bytes = 0, k0 = 0, k1 = 0;
    int tile[kMT];
    const lds_u8* row = lds;
    for (;;) {
#pragma unroll
      for (int slot = 0; slot < kRing; ++slot) {
        if (u == 0) {
          k0 = p.k_begin(item);
          k1 = min(k0 + len, K);
          if (p.group(item) != group) {
            group = p.group(item);
            const int rows = p.rows(group);
            barrier();  // the group before has been read
            fetch_x(k0, k1, rows, [&](int part, int m) { return p.row_at(group, part, m); });
            // (in so many words: the compiler would wait for them again, and for the
            // weights ahead, where the paths meet)
            wait_vmcnt<0>();
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
        // This unit has landed: only the loads of the units behind it, which are
        // the youngest, may be under way.
        wait_vmcnt<(kRing - 1) * kLoads>();
        Scales& b = scales[slot];
        const int kb = k0 + (u * kWK + wk) * kUnit;
        if (kb < k1) {
          uint32_t sc[kNT][4], zs[kNT][4];
#pragma unroll
          for (int h = 0; h < kBlocks; ++h) {
            if (h == 0 || kMode != kCoarse) {
              spread(b.s, h, sc);
              if constexpr (kW == kWInt4Z) spread(b.z, h, zs);
            }
            mul(ring + slot * kUnitBytes, h, sc, zs, row + 2 * (kb + 128 * h - k0), part_bytes, tile);
          }
        }
        const bool end = ++u == turns;
        if constexpr (kMode == kNone) {
          if (end) {
            const auto v = __builtin_amdgcn_permlane16_swap(b.s[0], b.s[0], false, false);
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
              for (int m = 0; m < kMT; ++m) acc[n][m] *= scale_of<kS>(v[n]);
          }
        }
        wait_lgkmcnt<0>();  // the slot has been read
        fetch(b, slot);
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
          sums[(((wave * kNT + n) * kMT + m) * 16 + 4 * g + e) * 16 + r] = acc[n][m][e];
    wait_lgkmcnt<0>();
    barrier();
  }
  // The sum over K of set wn's tile n.
  __device__ __forceinline__ float sum_of(int wn, int n, int m, int row, int col) const {
    float v = 0.0f;
#pragma unroll
    for (int q = 0; q < kWK; ++q)
      v += sums[((((wn * kWK + q) * kNT + n) * kMT + m) * 16 + row) * 16 + col];
    return v;
  }
};

}  // namespace detail
}  // namespace hipgemm
