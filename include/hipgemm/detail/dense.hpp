// Products of 16-bit operands, fp32 sums, with the epilogues of a feed-forward
// block, and the two products of its backward pass:
//
//   forward   z[m, n]  = sum_k x[m, k] w[n, k]            both along K
//   of x      dx[m, k] = sum_n dz[m, n] w[n, k]           w across its rows
//   of w      dw[n, k] = sum_m dz[m, n] x[m, k]           both across their rows
//
// One kernel body serves the three: C (M x N) = sum over K of A(m, k) B(n, k), each
// operand either in rows along K (kCol false: element (m, k) at m ld + k) or across
// (kCol true: at k ld + m).  Nothing is transposed in memory: tiles go to LDS as they
// lie, and an operand that lies across K is turned on its way from LDS to registers
// (ds_read_b64_tr_b16: sixteen lanes read four k of sixteen columns, and each gets
// one column's four).
//
// Work decomposition: one workgroup = 4 waves (one per SIMD), persistent over the
// tiles (tile_walk / grouped_tile, layout.hpp).  Wave w owns the BM / 2 x BN / 2 part
// (w / 2, w % 2) of a tile as FA x FB blocks of 16 x 16 (v_mfma_f32_16x16x32).
// kGated: of a tile's BN rows of B, half are gate rows and half the up rows of the
// same columns, interleaved so that each wave holds both sums of its columns and
// forms act(g) u from its own registers.
//
// A step is 64 elements of K: 128 bytes of a row, whole lines.  S stages of LDS
// hold steps, brought by DMA (buffer_load_dwordx4 ... lds) S steps ahead.  A step runs
// as two halves with a set of registers each:
//   half 0 of step k: MFMA of set 0 | read set 1: half 1 of step k
//   barrier: every wave's reads of step k are done, step k + 1 has landed
//   half 1 of step k: MFMA of set 1 | read set 0: half 0 of step k + 1,
//                                   | DMA of step k + S into step k's stage, the first half
//   half 0 of step k + 1            | the other half
// A CU takes in 64 bytes a cycle, which is as long as a step's MFMA in tiles of 128 x 128 and
// longer in smaller ones, and a wave that issues into a full queue waits: all of a step's DMA
// in half 1 made it the longer half (256 x 128, one workgroup alone at K 8192 89 us, spread 78;
// 2048 x 4096 x 4096 60.6 / 59.0).
// The sequence runs on across tiles: what lies past a tile's last step is the next
// tile's first.  Steps of a tile are padded to at least S (padding reads zeros).
//
// 256 x 256 tiles have room for two stages only, and a step's DMA (16 KiB of each wave's,
// 64 bytes a cycle) keep the memory path busy for half of its matrix instructions' time: all of
// them issued in half 1 have half a step to land, which is too little where operands come from
// memory (4096 x 4096 x 14336 341 us, with operands in the caches 314; by quarters 317, 315).
// There a step runs as four quarters, 4 x 4
// blocks by the whole step each, with one set of registers for each half of the rows (low,
// high) of A and B, read anew as soon as its second use is over, and a fourth of the DMA:
//   Q00: A low  x B low  | read B high of k     | DMA A low  of k + 2
//   Q01: A low  x B high | read A high of k     | DMA B low  of k + 2
//   Q10: A high x B low  | read A low  of k + 1 | DMA B high of k + 2
//   Q11: A high x B high | read B low  of k + 1 | DMA A high of k + 2
// Q00 and Q10 start with a barrier; what they and the quarter after read was fetched five or
// six quarters before, and what is fetched over was read two quarters before, across a
// barrier.  At each barrier the sixteen newest DMA may be in flight.
//
// K order inside a step: lane group g = lane / 16 takes the eight k from 16 g + 8 h in
// half h, in both layouts: slots 2 g + h of a row (layout.hpp: no bank conflicts), or
// the LDS rows 16 g + 8 h .. + 7 of an operand that lies across.  There the 16-byte
// slot s of row k is stored at s ^ col_xor(k): the four rows that sixteen lanes read
// and the next lane group's four lie in different banks.
//
// kSplit: work units are (tile, K-slice) pairs that write their fp32 sums to
// `partial`; k_dense_reduce adds them in order and finishes.
//
// Epilogue: two neighbouring blocks' sums change places between lane groups
// (v_permlane16_swap), so that a lane has eight columns of a row: bias, activation, residual
// and all stores go 16 bytes per lane, 64 bytes of a row side by side, at any address.
// Only where N ends inside a lane's eight columns they go one by one.
#pragma once

#include <utility>

#include "arch.hpp"
#include "decode.hpp"
#include "epilogue.hpp"
#include "layout.hpp"

namespace hipgemm {
namespace detail {

// kEpi: what the sums become.
constexpr int kEpiPlain = 0;     // stored
constexpr int kEpiLinear = 1;    // bias, pre, activation
constexpr int kEpiResidual = 2;  // and a residual
constexpr int kEpiGated = 3;     // bias, pre, activation, product

// What becomes of the sums (types: kOut*, kIn*; strides in elements).
struct DenseEpi {
  uint8_t* y;
  const uint8_t* bias;  // or null
  const uint8_t* r;     // residual or null
  uint8_t* pre;         // sums with bias, or null
  long long ldy, ldr, ldp;
  long long up;         // gated: columns from a gate sum to its up sum, in pre and bias
  int act, y_type, p_type, b_type, r_type;
};

struct DenseArgs {
  const uint8_t *a, *b;
  long long lda, ldb;  // bytes
  long long up;        // gated: bytes from a gate row of B to its up row
  int M, N, K;         // result rows and columns, and the sum's length
  int group_m;
  int slices, slice_steps;  // kSplit: K-slices of 64 slice_steps
  float* partial;           // slices x M x ldpart
  long long ldpart;
  int part_slices;          // slices of a part of dz (dense_slope_body), or 0: of the whole
  float part_scale;         // of a part's sums to those of the part before
  DenseEpi epi;
};

// Two products of one launch: `first` workgroups for x, the others for w.
struct DensePair {
  DenseArgs x, w;
  int first;
};

template <int BM, int BN, int S>
struct CfgDense {
  static constexpr int kBM = BM, kBN = BN, kStages = S;
  static constexpr int kBK = 64, kRow = 2 * kBK;  // elements, bytes of a step
  static constexpr int kWM = BM / 2, kWN = BN / 2;
  static constexpr int kFA = kWM / 16, kFB = kWN / 16;
  static constexpr int kAStage = kBM * kRow;
  static constexpr int kStage = (kBM + kBN) * kRow;
  static constexpr int kLdsBytes = S * kStage;
  // The schedule by quarter steps (dense_tile_body), for tiles whose registers and LDS
  // hold no more than a step and the next.
  static constexpr bool kQuarters = BM == 256 && BN == 256;
  static_assert(!kQuarters || S == 2, "two stages");
  static constexpr int kDmaA = BM / 32, kDmaB = BN / 32;  // per wave and step
  static constexpr int kDma = kDmaA + kDmaB;
  static_assert(kLdsBytes <= 160 * 1024, "LDS");
};

// ---- eight neighbouring elements, or one ------------------------------------

__device__ __forceinline__ float widen(uint32_t h, int type) {
  return type == kInBf16 ? __builtin_bit_cast(float, h << 16)
                         : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
// Rounded to the 16-bit type, to nearest even.
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, bool bf16) {
  return bf16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}
// Sixteen bytes at an address that is a multiple of an element (the memory system takes
// any; the type says so to the compiler).
struct __attribute__((packed, aligned(2))) Any16 {
  i32x4 v;
};
__device__ __forceinline__ i32x4 load16(const uint8_t* p) {
  return reinterpret_cast<const Any16*>(p)->v;
}
// Eight elements as they lie in memory: 16-bit ones in a, fp32 in a and b.
struct Raw8 {
  i32x4 a, b;
};
__device__ __forceinline__ Raw8 raw8(const uint8_t* p, long long at, int type) {
  if (type == kInF32) return Raw8{load16(p + 4 * at), load16(p + 4 * at + 16)};
  return Raw8{load16(p + 2 * at), i32x4{}};
}
__device__ __forceinline__ void widen8(const Raw8& r, int type, float (&v)[8]) {
  if (type == kInF32) {
    const f32x4 a = __builtin_bit_cast(f32x4, r.a), b = __builtin_bit_cast(f32x4, r.b);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t d = (uint32_t)r.a[e];
      if (type == kInBf16) {
        v[2 * e] = __builtin_bit_cast(float, d << 16);
        v[2 * e + 1] = __builtin_bit_cast(float, d & 0xffff0000u);
      } else {
        v[2 * e] = widen(d & 0xffffu, type);
        v[2 * e + 1] = widen(d >> 16, type);
      }
    }
  }
}
__device__ __forceinline__ void load8(const uint8_t* p, long long at, int type,
                                      float (&v)[8]) {
  widen8(raw8(p, at, type), type, v);
}
__device__ __forceinline__ float load1(const uint8_t* p, long long at, int type) {
  if (type == kInF32) return *reinterpret_cast<const float*>(p + 4 * at);
  return widen(*reinterpret_cast<const uint16_t*>(p + 2 * at), type);
}
// A store of 16 bytes, and the wait states of store_b128 (arch.hpp).
__device__ __forceinline__ void store16(uint8_t* p, i32x4 v) {
  reinterpret_cast<Any16*>(p)->v = v;
  asm volatile("s_nop 1" ::: "memory");
}
__device__ __forceinline__ void store8(uint8_t* p, long long at, int out,
                                       const float (&v)[8]) {
  if (out == kOutF32) {
    store16(p + 4 * at, __builtin_bit_cast(i32x4, f32x4{v[0], v[1], v[2], v[3]}));
    store16(p + 4 * at + 16, __builtin_bit_cast(i32x4, f32x4{v[4], v[5], v[6], v[7]}));
  } else {
    const bool b = out == kOutBf16;
    store16(p + 2 * at, i32x4{(int)narrow2(v[0], v[1], b), (int)narrow2(v[2], v[3], b),
                              (int)narrow2(v[4], v[5], b), (int)narrow2(v[6], v[7], b)});
  }
}
__device__ __forceinline__ void store1(uint8_t* p, long long at, int out, float v) {
  if (out == kOutF32) *reinterpret_cast<float*>(p + 4 * at) = v;
  else *reinterpret_cast<uint16_t*>(p + 2 * at) = (uint16_t)narrow2(v, 0.0f, out == kOutBf16);
}

__device__ __forceinline__ float activate(float v, int act) {
  return act == kActRelu       ? relu(v)
         : act == kActSilu     ? silu(v)
         : act == kActGeluTanh ? gelu_tanh(v)
                               : v;
}
__device__ __forceinline__ void activate8(float (&v)[8], int act) {
  if (act == kActRelu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = relu(v[e]);
  } else if (act == kActSilu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = silu(v[e]);
  } else if (act == kActGeluTanh) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = gelu_tanh(v[e]);
  }
}

// Element offsets of a row's first column here in the result, the residual and pre.
struct DenseAt {
  long long y, r, p;
};
__device__ __forceinline__ DenseAt dense_at(const DenseEpi& e, long long row, int col) {
  return DenseAt{row * e.ldy + col, row * e.ldr + col, row * e.ldp + col};
}

// Eight columns from `at` + c: v (gated: gate sums, u the up sums), with the bias; r: the
// residual, if there is one.
template <int kEpi>
__device__ __forceinline__ void finish8(const DenseEpi& e, const DenseAt& at, int c,
                                        float (&v)[8], float (&u)[8], const Raw8& r) {
  if constexpr (kEpi != kEpiPlain) {
    if (e.pre) {
      store8(e.pre, at.p + c, e.p_type, v);
      if constexpr (kEpi == kEpiGated) store8(e.pre, at.p + e.up + c, e.p_type, u);
    }
    activate8(v, e.act);
  }
  if constexpr (kEpi == kEpiGated) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= u[i];
  }
  if constexpr (kEpi == kEpiResidual) {
    float w[8];
    widen8(r, e.r_type, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += w[i];
  }
  store8(e.y, at.y + c, e.y_type, v);
}
// One column; v, u without the bias.
template <int kEpi>
__device__ __forceinline__ void finish1(const DenseEpi& e, const DenseAt& at, int c, int col,
                                        float v, float u) {
  if constexpr (kEpi != kEpiPlain) {
    if (e.bias) {
      v += load1(e.bias, col, e.b_type);
      if constexpr (kEpi == kEpiGated) u += load1(e.bias, e.up + col, e.b_type);
    }
    if (e.pre) {
      store1(e.pre, at.p + c, e.p_type, v);
      if constexpr (kEpi == kEpiGated) store1(e.pre, at.p + e.up + c, e.p_type, u);
    }
    v = activate(v, e.act);
  }
  if constexpr (kEpi == kEpiGated) v *= u;
  if constexpr (kEpi == kEpiResidual) v += load1(e.r, at.r + c, e.r_type);
  store1(e.y, at.y + c, e.y_type, v);
}

// ---- tiles --------------------------------------------------------------------

__host__ __device__ constexpr int col_xor(int k) { return 2 * ((k & 3) | (((k >> 4) & 1) << 2)); }

// f(0), .., f(N - 1) with constants.
template <int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
  [&]<int... I>(std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
  }(std::make_integer_sequence<int, N>{});
}
// Of `count` things spread evenly over `span` places from 0, those before place n.
constexpr int due(int n, int span, int count) {
  return n <= 0 ? 0 : n >= span ? count : (n * count + span - 1) / span;
}

using s16x4 = short __attribute__((ext_vector_type(4)));
using s16x8 = short __attribute__((ext_vector_type(8)));

// Sixteen lanes give the addresses of four columns' elements in each of four rows (lane
// i: row i / 4, columns 4 (i % 4) ..); lane i gets column i's four.  (__restrict: a
// read without any aliasing information is made to wait for every DMA in flight.)
__device__ __forceinline__ s16x4 lds_read_across(const lds_u8* __restrict p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4*)p);
}

// c += a b, in place.  Written as an instruction of its own: given the builtin, the
// register allocator moves accumulators about inside the K loop (36 to 180
// v_accvgpr_* of a step's 128 MFMA, 256 x 256 tiles).  The compiler does not see a matrix
// instruction here: operands are waited for (wait_lgkmcnt) before their first use, and
// mfma_drain() stands between the last one and the first read of a sum.
template <int kX>
__device__ __forceinline__ void mfma_acc(i32x4 a, i32x4 b, f32x4& c) {
  if constexpr (kX == kInBf16)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

template <class Cfg, int kX, bool kACol, bool kBCol, int kEpi, bool kSplit, bool kOnce = false>
__device__ __forceinline__ void dense_tile_body(const DenseArgs& g, lds_u8* lds, int block,
                                                int blocks) {
  constexpr bool kGated = kEpi == kEpiGated, kRes = kEpi == kEpiResidual;
  constexpr int S = Cfg::kStages, FA = Cfg::kFA, FB = Cfg::kFB;
  constexpr int kBK = Cfg::kBK, kDma = Cfg::kDma;
  constexpr int kMfma = FA * FB;  // of a half
  constexpr int kReadA = kACol ? 2 : 1, kReadB = kBCol ? 2 : 1;  // of a fragment
  constexpr int kReads = kReadA * FA + kReadB * FB;
  // MFMA of half 0 that are issued after the barrier: they read registers only and
  // keep the matrix unit busy while the waves meet.
  constexpr int kTail = kMfma >= 16 ? 2 : 0, kHead = kMfma - kTail;
  constexpr int kSpan = kMfma * 48 / 64;
  constexpr bool kQ = Cfg::kQuarters;
  constexpr int kWNr = kGated ? Cfg::kWN / 2 : Cfg::kWN;  // result columns of a wave
  constexpr int kBNr = 2 * kWNr;
  static_assert((S - 2) * kDma < 64, "vmcnt range");
  static_assert(!kGated || !kBCol, "gated: weights along K");
  const int lane = lane_id(), wave = wave_id();
  const int wm = wave >> 1, wn = wave & 1;
  const int tiles_m = (g.M + Cfg::kBM - 1) / Cfg::kBM;
  const int tiles_n = (g.N + kBNr - 1) / kBNr;
  const int tiles = tiles_m * tiles_n;
  const int units = kSplit ? tiles * g.slices : tiles;
  const int steps = kSplit ? g.slice_steps : (int)(((long long)g.K + kBK - 1) / kBK);
  const int steps_pad = max(S, steps);
  const TileWalk walk = tile_walk(block, blocks, units);
  int t = walk.first;
  if (t >= walk.end) return;

  // ---- DMA lane geometry -------------------------------------------------------
  // Along K: instruction q of wave w covers rows (4 q + w) 8 .. + 8, lane l row l / 8,
  // slot l % 8, which holds chunk (l % 8) ^ slot_xor(row).
  // Across: 1 KiB of rows of 2 BM bytes, lane l 16 bytes each; slot s of row k holds
  // the columns' chunk s ^ col_xor(k).
  const int drow = lane >> 3;
  const int dchunk = (lane & 7) ^ slot_xor(8 * (wave & 1) + drow);
  auto lane_off = [&](bool col, int width, long long ld, int q) -> uint32_t {
    if (!col) return (uint32_t)((4 * q + wave) * 8 + drow) * (uint32_t)ld + dchunk * 16;
    if constexpr (kQ) {  // two halves of the columns, below
      const int k = (4 * (q % 4) + wave) * 4 + lane / 16, c = (lane % 16) ^ col_xor(k);
      return (uint32_t)k * (uint32_t)ld + (c % 8 + 16 * (c / 8) + 8 * (q / 4)) * 16;
    }
    const int slots = width / 8, k = (4 * q + wave) * (64 / slots) + lane / slots;
    return (uint32_t)k * (uint32_t)ld + (((lane % slots) ^ col_xor(k)) * 16);
  };
  // Gated: row R of the tile's BN rows is column kWNr (R / kWN) + R % kWNr, of the up
  // half where R % kWN >= kWNr: whole instructions (eight rows) of one half.
  auto is_up = [&](int q) { return kGated && ((4 * q + wave) * 8) % Cfg::kWN >= kWNr; };
  uint32_t voff_a[Cfg::kDmaA], voff_b[Cfg::kDmaB];
#pragma unroll
  for (int q = 0; q < Cfg::kDmaA; ++q) voff_a[q] = lane_off(kACol, Cfg::kBM, g.lda, q);
#pragma unroll
  for (int q = 0; q < Cfg::kDmaB; ++q) {
    if constexpr (kGated) {
      const int R = (4 * q + wave) * 8;
      voff_b[q] = (uint32_t)(kWNr * (R / Cfg::kWN) + R % kWNr + drow) * (uint32_t)g.ldb +
                  dchunk * 16;
    } else {
      voff_b[q] = lane_off(kBCol, Cfg::kBN, g.ldb, q);
    }
  }

  // (Kept in registers: otherwise computed anew in every step.)
  auto keep = [&]() {
#pragma unroll
    for (int q = 0; q < Cfg::kDmaA; ++q) asm volatile("" : "+v"(voff_a[q]));
#pragma unroll
    for (int q = 0; q < Cfg::kDmaB; ++q) asm volatile("" : "+v"(voff_b[q]));
  };
  keep();
  // The same for a step that is not whole: offsets of lanes past the sum's end lie outside.
  // They change only where such a step comes or goes (2 % at 4096 x 4096 x 14336 against
  // a mask for every DMA).
  bool masked = false;
  auto mask = [&](uint32_t oob) {
    if constexpr (!kACol) {
#pragma unroll
      for (int q = 0; q < Cfg::kDmaA; ++q) voff_a[q] = (voff_a[q] & ~kOobOffset) | oob;
    }
    if constexpr (!kBCol) {
#pragma unroll
      for (int q = 0; q < Cfg::kDmaB; ++q) voff_b[q] = (voff_b[q] & ~kOobOffset) | oob;
    }
    keep();
  };

  // A unit's operands: along K the rows' resource; across, the columns' address, from
  // which each step's resource is made (rows past the sum's end read zero).
  struct Src {
    __amdgpu_buffer_rsrc_t a, b, b2;
    const uint8_t *pa, *pb;
    uint32_t ca, cb;  // across: bytes of a row from pa, pb
    int k0, kend;
    int full, rot;  // whole steps, and the one it starts at
  };
  auto rows_of = [](const uint8_t* p, long long ld, int first, int have, int most) {
    const int n = min(most, have - first);
    return make_rsrc(p + (long long)first * ld, (uint32_t)n * (uint32_t)ld);
  };
  auto src_of = [&](int unit) {
    Src s;
    if (unit >= walk.end) {
      s.a = s.b = s.b2 = make_rsrc(g.a, 0u);
      s.pa = s.pb = g.a;
      s.ca = s.cb = 0;
      s.k0 = s.kend = s.full = s.rot = 0;
      return s;
    }
    const int tile = kSplit ? unit % tiles : unit;
    const int slice = kSplit ? __builtin_amdgcn_readfirstlane(unit / tiles) : 0;
    const TileCoord c = grouped_tile_u(tile, tiles_m, tiles_n, g.group_m);
    const int m0 = c.m * Cfg::kBM, n0 = c.n * kBNr;
    s.k0 = kSplit ? slice * steps * kBK : 0;
    s.kend = kSplit ? (int)min((long long)g.K, (long long)s.k0 + (long long)steps * kBK) : g.K;
    s.full = max(0, s.kend - s.k0) / kBK;
    s.rot = (int)(((unsigned)block & 7u) * (unsigned)s.full / 8u);
    s.a = s.b = s.b2 = make_rsrc(g.a, 0u);
    s.pa = g.a;
    s.pb = g.b;
    s.ca = s.cb = 0;
    if constexpr (kACol) {
      s.pa = g.a + 2ll * m0;
      s.ca = (uint32_t)(2 * (((g.M + 7) & ~7) - m0));
    } else {
      s.a = rows_of(g.a, g.lda, m0, g.M, Cfg::kBM);
    }
    if constexpr (kBCol) {
      s.pb = g.b + 2ll * n0;
      s.cb = (uint32_t)(2 * (((g.N + 7) & ~7) - n0));
    } else {
      s.b = rows_of(g.b, g.ldb, n0, g.N, kBNr);
      if constexpr (kGated) s.b2 = rows_of(g.b + g.up, g.ldb, n0, g.N, kBNr);
    }
    return s;
  };
  Src cur = src_of(t), nxt = src_of(t + walk.stride);

  struct Step {
    __amdgpu_buffer_rsrc_t a, b, b2;
    uint32_t soff;
  };
  // Step d of the unit, or past its end step d - steps_pad of the next.
  auto step_src = [&](int d) {
    const bool next = d >= steps_pad;
    const int at = next ? d - steps_pad : d, full = next ? nxt.full : cur.full;
    int turned = at + (next ? nxt.rot : cur.rot);
    if (turned >= full) turned -= full;
    const int k = (next ? nxt.k0 : cur.k0) + (at < full ? turned : at) * kBK;
    const int kend = next ? nxt.kend : cur.kend;
    Step s;
    uint32_t soff = (uint32_t)k * 2u;
    asm volatile("" : "+s"(soff));
    s.soff = soff;
    if constexpr (!kACol || !kBCol) {
      if (at >= full || masked) {
        mask(k + dchunk * 8 < kend ? 0u : kOobOffset);
        masked = at >= full;
      }
    }
    auto across = [&](const uint8_t* p, long long ld, uint32_t cols) {
      const int rows = min(kBK, kend - k);
      return make_rsrc(p + (long long)k * ld,
                       rows > 0 ? (uint32_t)(rows - 1) * (uint32_t)ld + cols : 0u);
    };
    if constexpr (kACol) s.a = across(next ? nxt.pa : cur.pa, g.lda, next ? nxt.ca : cur.ca);
    else s.a = next ? nxt.a : cur.a;
    if constexpr (kBCol) s.b = across(next ? nxt.pb : cur.pb, g.ldb, next ? nxt.cb : cur.cb);
    else s.b = next ? nxt.b : cur.b;
    s.b2 = s.b;
    if constexpr (kGated) s.b2 = next ? nxt.b2 : cur.b2;
    return s;
  };
  auto dma_one = [&](const Step& s, int dst, int n) {
    const bool is_a = n < Cfg::kDmaA;
    const int q = is_a ? n : n - Cfg::kDmaA;
    lds_u8* to = lds + dst + (is_a ? 0 : Cfg::kAStage) + (4 * q + wave) * 1024;
    const uint32_t vo = is_a ? voff_a[q] : voff_b[q];
    const bool col = is_a ? kACol : kBCol;
    const uint32_t so = col ? 0u : s.soff;
    if (is_a) dma16(s.a, to, vo, so);
    else if (kOnce) dma16_nt(is_up(q) ? s.b2 : s.b, to, vo, so);
    else dma16(is_up(q) ? s.b2 : s.b, to, vo, so);
  };

  // ---- fragments ---------------------------------------------------------------
  const int r16 = lane & 15, grp = lane >> 4;
  // Along K: row r16 of the fragment, slot 2 grp + h.
  const uint32_t row_a = (uint32_t)((wm * Cfg::kWM + r16) * Cfg::kRow);
  const uint32_t row_b = (uint32_t)(Cfg::kAStage + (wn * Cfg::kWN + r16) * Cfg::kRow);
  uint32_t slot[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) slot[h] = (uint32_t)(((2 * grp + h) ^ slot_xor(r16)) * 16);
  // Across: LDS row 16 grp + 8 h + 4 p + r16 / 4, columns 16 f + 4 (r16 % 4) .. + 3.
  const int krow = 16 * grp + (r16 >> 2);
  const int kx = col_xor(krow);
  const uint32_t sub = (uint32_t)((((r16 & 3) >> 1) * 16) + (r16 & 1) * 8);
  // (By quarters: LDS rows of 128 columns, those of one half of both waves'.)
  constexpr int kParts = kQ ? 2 : 1, kCA = FA / kParts, kCB = FB / kParts;
  constexpr int kWideA = 2 * Cfg::kBM / kParts, kWideB = 2 * Cfg::kBN / kParts;
  uint32_t col_a[kCA], col_b[kCB];
#pragma unroll
  for (int f = 0; f < kCA; ++f)
    col_a[f] = (uint32_t)(krow * kWideA) + sub + (uint32_t)(((2 * (wm * kCA + f)) ^ kx) * 16);
#pragma unroll
  for (int f = 0; f < kCB; ++f)
    col_b[f] = (uint32_t)(Cfg::kAStage + krow * kWideB) + sub +
               (uint32_t)(((2 * (wn * kCB + f)) ^ kx) * 16);

  s16x4 fa[2][FA][2], fb[2][FB][2];
  // Fragment f of an operand, half h of the step in the stage at `st`, part p of it.
  auto read = [&](bool is_b, int st, int h, int f, int p) {
    s16x4(&to)[2] = is_b ? fb[h][f] : fa[h][f];
    if (is_b ? kBCol : kACol) {
      const int width = is_b ? kWideB : kWideA, c = f % (is_b ? kCB : kCA);
      const int part = f / (is_b ? kCB : kCA) * kBK * width;
      to[p] = lds_read_across(lds + st + (is_b ? col_b[c] : col_a[c]) + part +
                              (8 * h + 4 * p) * width);
    } else {
      const lds_u8* from = lds + st + (is_b ? row_b : row_a) + slot[h] + f * 16 * Cfg::kRow;
      const s16x8 v = __builtin_bit_cast(s16x8, lds_read16(from));
      to[0] = __builtin_shufflevector(v, v, 0, 1, 2, 3);
      to[1] = __builtin_shufflevector(v, v, 4, 5, 6, 7);
    }
  };
  // Read n of half h, in the order in which the MFMA need them: A 0, every B, the other A.
  auto read_one = [&](int st, int h, int n) {
    constexpr int kFirst = kReadA, kMid = kReadA + kReadB * FB;
    const bool is_b = n >= kFirst && n < kMid;
    const int m = is_b ? n - kFirst : n < kFirst ? n : n - kReadB * FB;
    const int per = is_b ? kReadB : kReadA;
    read(is_b, st, h, m / per, m % per);
  };
  auto frag = [](const s16x4 (&p)[2]) {
    return __builtin_bit_cast(i32x4, __builtin_shufflevector(p[0], p[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x4 acc[FA][FB];
  // Blocks row by row, odd rows right to left (neighbouring MFMA share an operand).
  auto mfma = [&](int h, int n) {
    const int i = n / FB, j = i % 2 ? FB - 1 - n % FB : n % FB;
    mfma_acc<kX>(frag(fb[h][j]), frag(fa[h][i]), acc[i][j]);
  };
  // Each MFMA of a half is followed by the reads and DMA that are due: reads spread over
  // three quarters of its MFMA, DMA over all (256 x 256 x K 14336 / 4096 by halves, both in rows,
  // TFLOP/s: 1552 / 1409; reads one after each of the first sixteen MFMA and DMA after them
  // 1543 / 1385, across K 1315 for 1410: bursts queue).
  // A step's DMA of which half 1 issues the first kFirst, and half 0 of the next the others.
  constexpr int kFirst = (kDma + 1) / 2, kRest = kDma - kFirst;
  Step src;
  auto half0 = [&](int st, int last) {
    wait_lgkmcnt<0>();
    static_for<kHead>([&](auto n) {
      mfma(0, n);
      static_for<due(n + 1, kSpan, kReads) - due(n, kSpan, kReads)>(
          [&](auto r) { read_one(st, 1, due(n, kSpan, kReads) + r); });
      static_for<due(n + 1, kHead, kRest) - due(n, kHead, kRest)>(
          [&](auto q) { dma_one(src, last, kFirst + due(n, kHead, kRest) + q); });
      sched_fence();
    });
  };
  auto half1 = [&](int st, int rst, int d) {
    src = step_src(d);
    static_for<kTail>([&](auto n) { mfma(0, kHead + n); });
    sched_fence();
    static_for<kMfma>([&](auto n) {
      mfma(1, n);
      static_for<due(n + 1, kSpan, kReads) - due(n, kSpan, kReads)>(
          [&](auto r) { read_one(rst, 0, due(n, kSpan, kReads) + r); });
      static_for<due(n + 1, kMfma, kFirst) - due(n, kMfma, kFirst)>(
          [&](auto q) { dma_one(src, st, due(n, kMfma, kFirst) + q); });
      sched_fence();
    });
  };
  auto next_stage = [](int s) {
    s += Cfg::kStage;
    return s == S * Cfg::kStage ? 0 : s;
  };
  int st = 0, last = (S - 1) * Cfg::kStage;
  bool stored = false;  // the previous tile was whole: all its stores were issued
  constexpr int kStores = FA * FB / (kGated ? 4 : 2);  // at least
  static_assert((S - 2) * kDma + kStores < 64, "vmcnt range");
  auto step_halves = [&](int k) {
    const int rst = next_stage(st);
    half0(st, last);
    // Step k + 1 has landed: newer are the DMA of S - 2 steps, and in a tile's first S - 2
    // steps the stores of the one before.
    wait_lgkmcnt<0>();
    if (stored && k < S - 2) wait_vmcnt<(S - 2) * kDma + kStores>();
    else wait_vmcnt<(S - 2) * kDma>();
    barrier();
    half1(st, rst, k + S);
    last = st;
    st = rst;
  };

  // ---- by quarters -------------------------------------------------------------
  constexpr int kQMfma = 32, kQTail = 2;
  static_assert(!kQ || (FA == 8 && FB == 8 && kDma == 16), "quarters of 4 x 4 blocks");
  auto mfma_q = [&](int qi, int qj, int n) {
    const int h = n / 16, i = n % 16 / 4, j = i % 2 ? 3 - n % 4 : n % 4;
    mfma_acc<kX>(frag(fb[h][4 * qj + j]), frag(fa[h][4 * qi + i]), acc[4 * qi + i][4 * qj + j]);
  };
  // Reads go with the first half of a quarter's matrix instructions, DMA with the second.
  // Blocks (qi, qj); reads of part rhi of operand rb (0: A, 1: B) from the stage at rst;
  // DMA of part dhi of operand db into the stage at dst.
  auto quarter = [&](int qi, int qj, auto rb, int rhi, int rst, auto db, int dhi, int dst,
                     const Step& src) {
    constexpr bool kRB = decltype(rb)::value, kDB = decltype(db)::value;
    constexpr int per = kRB ? kReadB : kReadA, reads = 8 * per;
    static_for<kQMfma - kQTail>([&](auto n) {
      mfma_q(qi, qj, n);
      static_for<due(n + 1, 16, reads) - due(n, 16, reads)>([&](auto r) {
        constexpr int x = due(n, 16, reads) + r;
        read(kRB, rst, x / per / 4, 4 * rhi + x / per % 4, x % per);
      });
      static_for<due(n - 15, 16, 4) - due(n - 16, 16, 4)>([&](auto d) {
        constexpr int x = due(n - 16, 16, 4) + d;
        const int q = (kDB ? kBCol : kACol) ? 4 * dhi + x : x % 2 + 4 * (x / 2) + 2 * dhi;
        dma_one(src, dst, kDB ? Cfg::kDmaA + q : q);
      });
      sched_fence();
    });
  };
  auto tail_q = [&](int qi, int qj) {
    static_for<kQTail>([&](auto n) { mfma_q(qi, qj, kQMfma - kQTail + n); });
    sched_fence();
  };
  auto step_quarters = [&](int k) {
    const std::false_type A{};
    const std::true_type B{};
    const int nst = next_stage(st);
    wait_lgkmcnt<0>();
    if (stored && k < 2) wait_vmcnt<16 + kStores>();
    else wait_vmcnt<16>();
    barrier();
    const Step src = step_src(k + 2);
    if (k > 0) tail_q(1, 1);
    quarter(0, 0, B, 1, st, A, 0, st, src);
    wait_lgkmcnt<0>();
    tail_q(0, 0);
    quarter(0, 1, A, 1, st, B, 0, st, src);
    wait_lgkmcnt<0>();
    if (stored && k == 0) wait_vmcnt<16 + kStores>();
    else wait_vmcnt<16>();
    barrier();
    tail_q(0, 1);
    quarter(1, 0, A, 0, nst, B, 1, st, src);
    wait_lgkmcnt<0>();
    tail_q(1, 0);
    quarter(1, 1, B, 0, nst, A, 1, st, src);
    st = nst;
  };

  if constexpr (kQ) {
    // In the order of the loop: A low, B low, B high, A high.
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const Step src = step_src(d);
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        const bool is_b = n >= 4 && n < 12;
        const int hi = n >= 8, x = n % 4;
        const int q = (is_b ? kBCol : kACol) ? 4 * hi + x : x % 2 + 4 * (x / 2) + 2 * hi;
        dma_one(src, d * Cfg::kStage, is_b ? Cfg::kDmaA + q : q);
      }
    }
    wait_vmcnt<16>();
    barrier();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int f = 0; f < 4; ++f) {
#pragma unroll
        for (int p = 0; p < kReadA; ++p) read(false, 0, h, f, p);
#pragma unroll
        for (int p = 0; p < kReadB; ++p) read(true, 0, h, f, p);
      }
  } else {
#pragma unroll
    for (int d = 0; d < S; ++d) {
      src = step_src(d);
#pragma unroll
      for (int n = 0; n < (d < S - 1 ? kDma : kFirst); ++n) dma_one(src, d * Cfg::kStage, n);
    }
    wait_vmcnt<(S - 2) * kDma + kFirst>();
    barrier();
#pragma unroll
    for (int n = 0; n < kReads; ++n) read_one(0, 0, n);
  }

  for (;;) {
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j) {
        acc[i][j] = f32x4{};
        asm volatile("" : "+a"(acc[i][j]));
      }
    // Two wait states from the last zero's write to the first matrix instruction.
    asm volatile("s_nop 3");
    if constexpr (kQ) {
      for (int k = 0; k < steps_pad; ++k) step_quarters(k);
      tail_q(1, 1);
    } else {
      for (int k = 0; k < steps_pad; ++k) step_halves(k);
    }

    // ---- epilogue --------------------------------------------------------------
    mfma_drain();
    const int tile = kSplit ? t % tiles : t;
    const TileCoord tc = grouped_tile_u(tile, tiles_m, tiles_n, g.group_m);
    const int row0 = tc.m * Cfg::kBM + wm * Cfg::kWM, col0 = tc.n * kBNr + wn * kWNr;
    int el = lane;
    asm volatile("" : "+v"(el));
    const DenseEpi& e = g.epi;
    stored = row0 + Cfg::kWM <= g.M && col0 + kWNr <= g.N;
    // The wave's part is whole and its results are of the operands' type (pre of fp32), which
    // is not asked again for every store (8192 x 8192 x 1024, relu: 147 / 130 us; gated 2048 x
    // 14336 x 4096 367 / 357).  With a residual it gained nothing and took scratch memory.
    constexpr bool kPlain = !kSplit && !kRes;
    constexpr int kOwnType = kX == kInBf16 ? kOutBf16 : kOutF16;
    const bool plain =
        kPlain && stored && e.y_type == kOwnType && (!e.pre || e.p_type == kOutF32);
    // Pair p of blocks: the lane's eight columns from col_l + 32 p (gated: of the gate where
    // p < kResults, of the up half after).
    constexpr int kPairs = FB / 2, kResults = kGated ? kPairs / 2 : kPairs;
    int row_l = row0 + (el & 15);
    int col_l = col0 + 16 * ((el >> 4) & 1) + 8 * (el >> 5);
    auto whole = [&](int p) { return col_l + 32 * p + 8 <= g.N; };
    float bias[kPairs][8] = {};
    const bool biased = !kSplit && kEpi != kEpiPlain && e.bias;
    if (biased) {
#pragma unroll
      for (int p = 0; p < kPairs; ++p)
        if (whole(p % kResults))
          load8(e.bias, (p / kResults) * e.up + col_l + 32 * (p % kResults), e.b_type, bias[p]);
      // No load may look pending where the K loop starts again: the compiler would have
      // every step wait for all DMA before it uses the register.
#pragma unroll
      for (int p = 0; p < kPairs; ++p)
#pragma unroll
        for (int x = 0; x < 8; ++x) asm volatile("" : "+v"(bias[p][x]));
    }
    Raw8 res[kResults] = {};
    auto residual = [&](int row, long long at, int p) {
      if (row < g.M && whole(p)) res[p] = raw8(e.r, at + 32 * p, e.r_type);
    };
    if constexpr (kRes) {
#pragma unroll
      for (int p = 0; p < kResults; ++p) residual(row_l, row_l * e.ldr + col_l, p);
    }
    // (Rolled, the accumulators picked by branches: unrolled the epilogue is FA times
    // the code, and its array stays in memory.)
#pragma nounroll
    for (int i = 0; i < FA; ++i) {
      f32x4 blk[FB];
#pragma unroll
      for (int b = 0; b < FA; ++b)
        if (b == i) {
          // (Opaque: their elements are read here, not ahead of the loop, where nothing
          // would keep the reads behind mfma_drain.)
#pragma unroll
          for (int j = 0; j < FB; ++j) asm volatile("" : "+a"(acc[b][j]));
#pragma unroll
          for (int j = 0; j < FB; ++j) blk[j] = acc[b][j];
        }
      // Lane group g has columns 4 g .. + 3 of two neighbouring blocks; after the swap
      // of its odd 16 lanes with the other's even ones, eight of one block.
      float v[kPairs][8];
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
        // (Bit casts of whole vectors: of one element they yield element 0.)
        const i32x4 b0 = __builtin_bit_cast(i32x4, blk[2 * p]);
        const i32x4 b1 = __builtin_bit_cast(i32x4, blk[2 * p + 1]);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const auto s2 =
              __builtin_amdgcn_permlane16_swap((uint32_t)b0[x], (uint32_t)b1[x], false, false);
          const uint32_t lo = s2[0], hi = s2[1];
          v[p][x] = __builtin_bit_cast(float, lo);
          v[p][4 + x] = __builtin_bit_cast(float, hi);
        }
      }
      // (Opaque: addresses are made here, not all of them before the loop.)
      asm volatile("" : "+v"(row_l), "+v"(col_l));
      auto with_bias = [&](int p) {
        if (!biased) return;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          v[p][x] += bias[p][x];
          if constexpr (kGated) v[p + kResults][x] += bias[p + kResults][x];
        }
      };
      if (plain) {
        if constexpr (kPlain) {
          DenseEpi own = e;
          own.y_type = kOwnType;
          own.p_type = kOutF32;
          const DenseAt at = dense_at(own, row_l, col_l);
#pragma unroll
          for (int p = 0; p < kResults; ++p) {
            with_bias(p);
            finish8<kEpi>(own, at, 32 * p, v[p], v[kGated ? p + kResults : p], res[p]);
          }
        }
      } else if (row_l < g.M) {
        const DenseAt at = dense_at(e, row_l, col_l);
        const long long part =
            ((long long)(kSplit ? t / tiles : 0) * g.M + row_l) * g.ldpart + col_l;
#pragma unroll
        for (int p = 0; p < kResults; ++p) {
          const int col = col_l + 32 * p;
          float(&u)[8] = v[kGated ? p + kResults : p];
          if constexpr (kSplit) {
            if (col < g.N) {
              uint8_t* to = reinterpret_cast<uint8_t*>(g.partial);
              store8(to, part + 32 * p, kOutF32, v[p]);
              if constexpr (kGated) store8(to, part + g.ldpart / 2 + 32 * p, kOutF32, u);
            }
          } else if (whole(p)) {
            with_bias(p);
            finish8<kEpi>(e, at, 32 * p, v[p], u, res[p]);
            if (kRes && i + 1 < FA) residual(row_l + 16, at.r + 16 * e.ldr, p);
          } else {
#pragma unroll
            for (int x = 0; x < 8; ++x)
              if (col + x < g.N) finish1<kEpi>(e, at, 32 * p + x, col + x, v[p][x], u[x]);
          }
        }
      }
      row_l += 16;
    }
    // (As for the bias.)
    if constexpr (kRes) wait_vmcnt<0>();
    t += walk.stride;
    if (t >= walk.end) break;
    cur = nxt;
    nxt = src_of(t + walk.stride);
  }
  // The look-ahead's DMA (empty ranges) still write LDS.
  wait_vmcnt<0>();
}

// ---- K-slices' sums -----------------------------------------------------------

// A thread per row and eight columns: slices in order, then the epilogue.  Where the slices
// are those of dz's parts, each part's sums count part_scale of the one before; an infinite or
// NaN sum of the first part is the result (rests of zero times an infinite operand are NaN).
template <int kEpi>
__device__ __forceinline__ void dense_reduce_body(const DenseArgs& g) {
  constexpr bool kGated = kEpi == kEpiGated;
  const int units = (g.N + 7) / 8;
  const long long x = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long row = x / units;
  const int col = 8 * (int)(x % units);
  if (row >= g.M) return;
  float v[8] = {}, u[8] = {};
  const uint8_t* p = reinterpret_cast<const uint8_t*>(g.partial);
  float scale = 1.0f;
  bool finite[8] = {};
  for (int s = 0; s < g.slices; ++s) {
    const long long o = ((long long)s * g.M + row) * g.ldpart + col;
    float w[8];
    load8(p, o, kInF32, w);
    if constexpr (kEpi == kEpiPlain) {
      if (g.part_slices && s && s % g.part_slices == 0) {
        if (s == g.part_slices) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            finite[e] = __builtin_fabsf(v[e]) < __builtin_inff();
        }
        scale *= g.part_scale;
      }
      if (g.part_slices) {
        const bool rest = s >= g.part_slices;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          w[e] = rest && !finite[e] ? 0.0f : w[e] * scale;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += w[e];
    if constexpr (kGated) {
      load8(p, o + g.ldpart / 2, kInF32, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] += w[e];
    }
  }
  const DenseEpi& e = g.epi;
  const DenseAt at = dense_at(e, row, col);
  if (col + 8 <= g.N) {
    if (kEpi != kEpiPlain && e.bias) {
      float b[8];
      load8(e.bias, col, e.b_type, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += b[i];
      if constexpr (kGated) {
        load8(e.bias, e.up + col, e.b_type, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] += b[i];
      }
    }
    Raw8 r{};
    if constexpr (kEpi == kEpiResidual) r = raw8(e.r, at.r, e.r_type);
    finish8<kEpi>(e, at, 0, v, u, r);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < g.N) finish1<kEpi>(e, at, i, col + i, v[i], u[i]);
  }
}

// ---- gradients of the sums ----------------------------------------------------

// The activation's derivative at z, its limits at infinities (NaN stays NaN):
//   relu  z > 0
//   silu  s (1 + z (1 - s)),            s = 1 / (1 + e^-z)
//   gelu  s (1 + z (1 - s) 2 u'(z)),    s = 1 / (1 + e^(-2 u)),
//         u' = sqrt(2/pi) (1 + 3 0.044715 z^2)
// with z held to +-96 in the second factors, past which s or 1 - s is zero in fp32.
__device__ __forceinline__ float slope(float z, int act) {
  if (act == kActRelu) return z > 0.0f ? 1.0f : z != z ? z : 0.0f;
  if (act == kActNone) return 1.0f;
  const float c = __builtin_fminf(__builtin_fmaxf(z, -96.0f), 96.0f);
  float s, d = c;
  if (act == kActSilu) {
    s = __builtin_amdgcn_rcpf(1.0f + exp_fast(-c));
  } else {
    constexpr float k = 0.7978845608028654f;
    const float c2 = c * c;
    const float u2 = 2.0f * k * c * __builtin_fmaf(c2, 0.044715f, 1.0f);
    s = __builtin_amdgcn_rcpf(1.0f + exp_fast(-u2));
    d = 2.0f * k * c * __builtin_fmaf(c2, 3.0f * 0.044715f, 1.0f);
  }
  return z != z ? z : s * __builtin_fmaf(d, 1.0f - s, 1.0f);
}

constexpr int kSlopeColumns = 256;  // of a workgroup
struct SlopeArgs {
  const uint8_t *dy, *pre;
  uint8_t* dz;     // or null
  float* columns;  // gridDim.y x width sums of dz over a block's rows, or null
  long long lddy, ldp, lddz;
  int M, N;        // of dy; dz has 2 N columns where gated
  int act, dy_type, p_type;
  int rows;        // of a block
  int parts;       // of dz: matrices of `plane` elements
  long long plane;
};

// What rounding to the operands' type left of v, times kRest (one that is infinite or NaN
// leaves nothing).  Rests of fp16 values are scaled into its range.
template <int kX>
constexpr float kRest = kX == kInBf16 ? 1.0f : 2048.0f;
template <int kX>
__device__ __forceinline__ void rest8(float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint32_t d = narrow2(v[e], v[e + 1], kX == kInBf16);
    const float lo = v[e] - widen(d & 0xffffu, kX), hi = v[e + 1] - widen(d >> 16, kX);
    v[e] = __builtin_fabsf(lo) < __builtin_inff() ? lo * kRest<kX> : 0.0f;
    v[e + 1] = __builtin_fabsf(hi) < __builtin_inff() ? hi * kRest<kX> : 0.0f;
  }
}

// dz = dy act'(z);  gated, z = [g | u]: [dy u act'(g) | dy act(g)].  Rounded to the
// operands' type, as the matrix instructions take it: half a step of every term of dx and dw,
// which are rounded to that type themselves.  For float32 results dz has further parts, each
// the rest that rounding the one before left, to 24 bits (bf16: three parts, fp16: two), and
// the products are sums over them (4096 x 16384 x 4096 bf16, dx and dw: 916 us, with dw in
// float32 1938).  Column sums are of the values before rounding, in fp32.
// A thread has eight columns and every eighth row of the block's.
// Columns from N to the padded row's end are written as zeros.
template <int kX, bool kGated>
__device__ __forceinline__ void dense_slope_body(const SlopeArgs& g, float* sums) {
  constexpr int kParts = kGated ? 2 : 1;
  constexpr int kOut = kX == kInBf16 ? kOutBf16 : kOutF16;
  constexpr int kTx = kSlopeColumns / 8, kTy = 256 / kTx;
  const int tx = threadIdx.x % kTx, ty = threadIdx.x / kTx;
  const int col = 8 * (kTx * blockIdx.x + tx);
  const long long first = (long long)blockIdx.y * g.rows;
  const long long end = min((long long)g.M, first + g.rows);
  const bool live = col < g.N;
  const bool whole = col + 8 <= g.N;
  float sum[kParts][8] = {};
  struct Row {
    Raw8 dy, z, u;
  };
  auto fetch = [&](long long row) {
    Row r{};
    if (whole) {
      r.dy = raw8(g.dy, row * g.lddy + col, g.dy_type);
      if (g.pre) r.z = raw8(g.pre, row * g.ldp + col, g.p_type);
      if constexpr (kGated) r.u = raw8(g.pre, row * g.ldp + g.N + col, g.p_type);
    }
    return r;
  };
  auto store = [&](long long at, float (&v)[8]) {
    store8(g.dz, at, kOut, v);
    for (int p = 1; p < g.parts; ++p) {
      rest8<kX>(v);
      store8(g.dz, p * g.plane + at, kOut, v);
    }
  };
  auto finish = [&](long long row, const Row& r) {
    float dy[8] = {}, z[8] = {}, u[8] = {};
    if (whole) {
      widen8(r.dy, g.dy_type, dy);
      if (g.pre) widen8(r.z, g.p_type, z);
      if constexpr (kGated) widen8(r.u, g.p_type, u);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < g.N) {
          dy[e] = load1(g.dy, row * g.lddy + col + e, g.dy_type);
          if (g.pre) z[e] = load1(g.pre, row * g.ldp + col + e, g.p_type);
          if constexpr (kGated) u[e] = load1(g.pre, row * g.ldp + g.N + col + e, g.p_type);
        }
    }
    float d[8];
    if constexpr (kGated) {
      float a[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        d[e] = dy[e] * u[e] * slope(z[e], g.act);
        a[e] = z[e];
      }
      activate8(a, g.act);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a[e] *= dy[e];
        sum[kParts - 1][e] += a[e];
      }
      if (g.dz) store(row * g.lddz + g.N + col, a);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = dy[e] * slope(z[e], g.act);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[0][e] += d[e];
    if (g.dz) store(row * g.lddz + col, d);
  };
  if (live)
    for (long long row = first + ty; row < end; row += kTy) finish(row, fetch(row));
  if (!g.columns) return;
  // The block's sums of each column, in order.
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[ty * kSlopeColumns + 8 * tx + e] = sum[p][e];
    __syncthreads();
    for (int x = threadIdx.x; x < kSlopeColumns; x += 256) {
      const int c = kSlopeColumns * blockIdx.x + x;
      float s = 0.0f;
#pragma unroll
      for (int y = 0; y < kTy; ++y) s += sums[y * kSlopeColumns + x];
      if (c < g.N) g.columns[((long long)blockIdx.y * kParts + p) * g.N + c] = s;
    }
  }
}

// out[c] = sum over blocks of columns[b][c]: sixteen columns of a workgroup, a sixteenth of
// the blocks each thread, whose sums are added in order.
__device__ __forceinline__ void dense_columns_body(const float* columns, int blocks, int N,
                                                   uint8_t* out, int type, float* sums) {
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, c = 16 * blockIdx.x + tx;
  float s = 0.0f;
  if (c < N)
#pragma unroll 4
    for (int b = ty; b < blocks; b += 16) s += columns[(long long)b * N + c];
  sums[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x >= 16 || c >= N) return;
#pragma unroll
  for (int y = 1; y < 16; ++y) s += sums[16 * y + tx];
  store1(out, c, type, s);
}

}  // namespace detail
}  // namespace hipgemm
