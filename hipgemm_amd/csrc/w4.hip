// hipgemm_w4_gemm: arguments, the choice of kernel and its launch.
#include "hipgemm.h"

#include "kernels.hpp"

#include "hipgemm/detail/w4_tile.hpp"

namespace hipgemm {
namespace kernels {

#define HIPGEMM_W4(X, W)                      \
  const void* w4_vec_##X##_##W(int s, int rows, int lk); \
  const void* w4_tile_##X##_##W(int s, int mode); \
  const void* w4_split_##X##_##W(int s, int mode, int mt, int nt);
HIPGEMM_W4(bf16, int4)
HIPGEMM_W4(bf16, int4z)
HIPGEMM_W4(bf16, fp4)
HIPGEMM_W4(f16, int4)
HIPGEMM_W4(f16, int4z)
HIPGEMM_W4(f16, fp4)
#undef HIPGEMM_W4

const void* w4_vec(int x, int w, int s, int rows, int lk) {
  const bool b = x == detail::kInBf16;
  switch (w) {
    case detail::kWInt4: return b ? w4_vec_bf16_int4(s, rows, lk) : w4_vec_f16_int4(s, rows, lk);
    case detail::kWInt4Z: return b ? w4_vec_bf16_int4z(s, rows, lk) : w4_vec_f16_int4z(s, rows, lk);
    default: return b ? w4_vec_bf16_fp4(s, rows, lk) : w4_vec_f16_fp4(s, rows, lk);
  }
}
const void* w4_tile(int x, int w, int s, int mode) {
  const bool b = x == detail::kInBf16;
  switch (w) {
    case detail::kWInt4: return b ? w4_tile_bf16_int4(s, mode) : w4_tile_f16_int4(s, mode);
    case detail::kWInt4Z: return b ? w4_tile_bf16_int4z(s, mode) : w4_tile_f16_int4z(s, mode);
    default: return b ? w4_tile_bf16_fp4(s, mode) : w4_tile_f16_fp4(s, mode);
  }
}
const void* w4_split(int x, int w, int s, int mode, int mt, int nt) {
  const bool b = x == detail::kInBf16;
  switch (w) {
    case detail::kWInt4:
      return b ? w4_split_bf16_int4(s, mode, mt, nt) : w4_split_f16_int4(s, mode, mt, nt);
    case detail::kWInt4Z:
      return b ? w4_split_bf16_int4z(s, mode, mt, nt) : w4_split_f16_int4z(s, mode, mt, nt);
    default: return b ? w4_split_bf16_fp4(s, mode, mt, nt) : w4_split_f16_fp4(s, mode, mt, nt);
  }
}

}  // namespace kernels
}  // namespace hipgemm

namespace {

using namespace hipgemm::detail;
namespace hk = hipgemm::kernels;

static_assert(HIPGEMM_IN_F32 == kInF32 && HIPGEMM_IN_BF16 == kInBf16 &&
                  HIPGEMM_IN_F16 == kInF16 && HIPGEMM_SCALE_E8M0 == kScaleE8M0 &&
                  HIPGEMM_W4_INT4 == kWInt4 && HIPGEMM_W4_FP4 == kWFp4,
              "codes");

bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

constexpr int kMaxK = 1 << 26;
constexpr long long kMaxTileRow = 1 << 23;  // 128 rows' bytes in a buffer's range
constexpr long long kMaxRow = 1 << 25;      // 64 rows' bytes in a buffer's range

template <class Args>
hipError_t launch(const void* fn, dim3 grid, int threads, Args& g, hipStream_t stream) {
  if (!fn) return hipErrorInvalidValue;
  void* args[] = {&g};
  return hipLaunchKernel(fn, grid, dim3((unsigned)threads), args, 0, stream);
}

// k_w4_split: groups of up to 64 rows of even lengths, and 32 columns where that
// leaves a workgroup for each CU (16 rows, 4096 x 4096: 9.8 us for 13.4;  14336 x
// 4096, 448 tiles: 19.6 for 16.0).  Groups are halved while each CU still takes at
// most one such tile: weights are decoded once more, by CUs that had nothing to do
// (us, not halved / halved, int4: 64 x 256 x 8192 24.0/13.8, 256 x 512 x 8192
// 25.3/16.3, 37 x 2048 x 4096 12.1/9.5, 64 x 4096 x 4096 16.3/13.0, 703 x 256 x 22144
// 105/70, 128 x 512 x 512 6.5/4.8;  fp4 512 x 512 x 4096 15.9/12.9).  Groups of 48 rows
// beside those of 32 and 64 (us, 48 / 64): int4 37 x 5000 x 3584 12.4/14.5, in groups of
// 64 18.7/22.5, 48 x 14336 x 4096 20.2/22.3, 90 x 14336 x 4096 34.6/40.3; 40 x 4096 x 4096,
// halved to 32, alike.
struct SplitPlan {
  int mt, nt;
  long long tiles;
};
SplitPlan split_plan(int M, int N) {
  SplitPlan p;
  const int groups = (M + 63) / 64;
  p.mt = ((M + groups - 1) / groups + 15) / 16;
  auto groups_of = [M](int mt) { return (long long)((M + 16 * mt - 1) / (16 * mt)); };
  const long long narrow = (N + 31) / 32;
  while (p.mt > 1 && groups_of((p.mt + 1) / 2) * narrow <= 256) p.mt = (p.mt + 1) / 2;
  const long long tm = groups_of(p.mt);
  p.nt = tm * narrow <= 256 ? 2 : 4;
  p.tiles = tm * ((N + 16 * p.nt - 1) / (16 * p.nt));
  return p;
}

// Tiles of 128 x 128 where the split kernel's take four rounds over the CUs, five where
// the large ones are more than a workgroup per CU, and not of fewer rows than three
// quarters of a tile.  us in a graph, split / tile, K = 4096 but as given:
//   int4 in groups of 128
//     rounds 3: 129 x 14336 48/62, 192 x 14336 60/63, 300 x 8192 x 8192 99/108, 384 102/107
//     rounds 4: 97 x 28672 79/62, 256 x 14336 77/62, 1024 x 4096 83/63; 258 large tiles:
//       129 x 16600 63/86
//     rounds 5: 300 x 14336 95/86, 700 x 6144 98/86, 800 x 5000 x 3584 87/77
//     more: 512 x 14336 135/90, 2048 x 4096 188/96
//   int4 in groups of 32 with zero points: 129 x 14336 95/118, 192 117/118, 256 154/119
//   fp4, E8M0: 192 x 14336 56/64, 256 x 12288 56/64, 256 x 14336 69/64
//   three quarters of a tile: 96 x 28672 x 8192 112/109 (128: 131/115)
bool by_tiles(const hipgemm_w4_desc& d, const SplitPlan& p) {
  const long long tiles = (long long)((d.M + kW4TileM - 1) / kW4TileM) *
                          ((d.N + kW4TileN - 1) / kW4TileN);
  return d.M > 96 && p.tiles > 256 * (tiles <= 256 ? 3 : 4) && 2 * d.ldx <= kMaxTileRow &&
         d.ldw <= kMaxTileRow && d.lds <= kMaxTileRow;
}

// k_w4_vec: lanes of a row, and the waves along K and rows of a workgroup.
// 16 lanes where 64 would be idle for the most part.
struct VecPlan {
  int lk, waves_k, waves_r, rows, wave_rows;
};
VecPlan vec_plan(int N, int K) {
  VecPlan p;
  const int units = K / 32;
  p.lk = units > 24 ? 64 : 16;
  const int chunks = units > p.lk ? (units + p.lk - 1) / p.lk : 1;
  const int turns = (chunks + 7) / 8;
  p.waves_k = (chunks + turns - 1) / turns;
  p.waves_r = p.waves_k >= 4 ? 1 : 4 / p.waves_k;
  // Rows: two workgroups per CU, in whole steps of the waves.
  const int step = kVecRows * (kWave / p.lk);
  int steps = (N + 512 * step * p.waves_r - 1) / (512 * step * p.waves_r);
  if (steps * step > kVecMaxRows) steps = kVecMaxRows / step;
  p.wave_rows = steps * step;
  p.rows = p.wave_rows * p.waves_r;
  return p;
}

// The kernel of a call, and of tiles their rows and columns: vectors up to four rows;
// and, four at a time, without any K or where rows of x lie so far apart that 64 are
// not in a buffer's range.
hipgemm_w4_plan plan_of(const hipgemm_w4_desc& d) {
  if (d.M <= 4 || d.K == 0 || 2 * d.ldx > kMaxRow) return {HIPGEMM_W4_VECTORS, 0, 0};
  const SplitPlan p = split_plan(d.M, d.N);
  if (by_tiles(d, p)) return {HIPGEMM_W4_TILES, kW4TileM, kW4TileN};
  return {HIPGEMM_W4_SPLIT, 16 * p.mt, 16 * p.nt};
}

hipError_t run(const hipgemm_w4_desc& d, hipStream_t stream) {
  W4Args g{};
  g.x = static_cast<const uint8_t*>(d.x);
  g.w = static_cast<const uint8_t*>(d.weight);
  g.s = static_cast<const uint8_t*>(d.scales);
  g.z = d.zeros;
  g.y = static_cast<uint8_t*>(d.y);
  g.bias = d.bias;
  g.ldx = 2 * d.ldx;
  g.ldw = d.ldw;
  g.lds = d.lds * type_bytes(d.scale_type);
  g.ldz = d.lds;
  g.ldy = d.ldy;
  g.M = d.M;
  g.N = d.N;
  g.K = d.K;
  g.G = d.group_size;
  g.act = d.activation;
  g.out = d.out_dtype;
  const int w = d.zeros ? kWInt4Z : d.format;
  const hipgemm_w4_plan plan = plan_of(d);
  if (plan.kernel == HIPGEMM_W4_VECTORS) {
    const VecPlan p = vec_plan(d.N, d.K);
    g.waves_k = p.waves_k;
    g.rows = p.rows;
    g.wave_rows = p.wave_rows;
    for (int m = 0; m < d.M; m += 4) {
      g.M = d.M - m < 4 ? d.M - m : 4;
      const hipError_t e =
          launch(hk::w4_vec(d.x_type, w, d.scale_type, g.M == 3 ? 4 : g.M, p.lk),
                 dim3((unsigned)((d.N + p.rows - 1) / p.rows)), kWave * p.waves_k * p.waves_r, g,
                 stream);
      if (e != hipSuccess) return e;
      g.x += 4 * g.ldx;
      g.y += 4 * d.ldy * out_bytes(d.out_dtype);
    }
    return hipSuccess;
  }
  const int mode = d.format == HIPGEMM_W4_FP4 && d.scale_type == HIPGEMM_SCALE_E8M0 &&
                           d.x_type == HIPGEMM_IN_BF16
                       ? kInline
                   : d.group_size % 128 == 0 ? kCoarse
                                             : kFine;
  const long long tiles = (long long)((d.M + plan.tile_rows - 1) / plan.tile_rows) *
                          ((d.N + plan.tile_columns - 1) / plan.tile_columns);
  const bool by = plan.kernel == HIPGEMM_W4_TILES;
  const long long most = by ? 512 : 256;  // workgroups: two per CU, one
  const void* fn = by ? hk::w4_tile(d.x_type, w, d.scale_type, mode)
                      : hk::w4_split(d.x_type, w, d.scale_type, mode, plan.tile_rows / 16,
                                     plan.tile_columns / 16);
  return launch(fn, dim3((unsigned)(tiles < most ? tiles : most)), 256, g, stream);
}

hipError_t check(const hipgemm_w4_desc* desc) {
  if (!desc || desc->size != sizeof(hipgemm_w4_desc)) return hipErrorInvalidValue;
  const hipgemm_w4_desc& d = *desc;
  if (d.M < 0 || d.N < 0 || d.K < 0 || d.K % 32 != 0 || d.K > kMaxK || d.group_size <= 0 ||
      d.group_size % 32 != 0)
    return hipErrorInvalidValue;
  if ((d.x_type != HIPGEMM_IN_BF16 && d.x_type != HIPGEMM_IN_F16) ||
      (d.format != HIPGEMM_W4_INT4 && d.format != HIPGEMM_W4_FP4) || d.scale_type < 0 ||
      d.scale_type > HIPGEMM_SCALE_E8M0 || d.out_dtype < 0 || d.out_dtype > HIPGEMM_OUT_F32 ||
      d.activation < 0 || d.activation > HIPGEMM_ACT_SILU ||
      (d.format == HIPGEMM_W4_FP4 && d.zeros))
    return hipErrorInvalidValue;
  if (d.M == 0 || d.N == 0) return hipSuccess;
  if (!d.y || !aligned(d.y, out_bytes(d.out_dtype)) || d.ldy < d.N ||
      (d.bias && !aligned(d.bias, 4)))
    return hipErrorInvalidValue;
  if (d.K > 0) {
    if (!d.x || !d.weight || !d.scales || !aligned(d.x, 16) || !aligned(d.weight, 16) ||
        !aligned(d.scales, type_bytes(d.scale_type)))
      return hipErrorInvalidValue;
    if (d.ldx < d.K || d.ldx % 8 != 0 || d.ldw < d.K / 2 || d.ldw % 16 != 0 ||
        d.ldw > kMaxRow || d.lds > kMaxRow / type_bytes(d.scale_type) ||
        d.lds < (d.K - 1) / d.group_size + 1)
      return hipErrorInvalidValue;
  }
  return hipSuccess;
}

}  // namespace

extern "C" hipError_t hipgemm_w4_gemm(const hipgemm_w4_desc* desc, hipStream_t stream) {
  const hipError_t e = check(desc);
  return e != hipSuccess || desc->M == 0 || desc->N == 0 ? e : run(*desc, stream);
}

extern "C" hipError_t hipgemm_w4_select(const hipgemm_w4_desc* desc, hipgemm_w4_plan* plan) {
  const hipError_t e = check(desc);
  if (e != hipSuccess || !plan) return hipErrorInvalidValue;
  *plan = plan_of(*desc);
  return hipSuccess;
}
