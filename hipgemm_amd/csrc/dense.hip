// hipgemm_linear and hipgemm_linear_backward: arguments, the choice of tiles, launches.
#include "hipgemm.h"

#include "kernels.hpp"

#include "hipgemm/detail/dense.hpp"

namespace hipgemm {
namespace kernels {

#define HIPGEMM_DENSE(L)                             \
  const void* dense_tile_bf16_##L(int tile, int mode); \
  const void* dense_tile_f16_##L(int tile, int mode);
HIPGEMM_DENSE(nt)
HIPGEMM_DENSE(res)
HIPGEMM_DENSE(nn)
HIPGEMM_DENSE(tn)
HIPGEMM_DENSE(gated)
#undef HIPGEMM_DENSE

const void* dense_pair_bf16();
const void* dense_pair_f16();
const void* dense_pair(int x) {
  return x == detail::kInBf16 ? dense_pair_bf16() : dense_pair_f16();
}

const void* dense_tile(int x, int kind, int tile, int mode) {
  const bool b = x == detail::kInBf16;
  switch (kind) {
    case kDenseNT: return b ? dense_tile_bf16_nt(tile, mode) : dense_tile_f16_nt(tile, mode);
    case kDenseRes: return b ? dense_tile_bf16_res(tile, mode) : dense_tile_f16_res(tile, mode);
    case kDenseNN: return b ? dense_tile_bf16_nn(tile, mode) : dense_tile_f16_nn(tile, mode);
    case kDenseTN: return b ? dense_tile_bf16_tn(tile, mode) : dense_tile_f16_tn(tile, mode);
    default:
      return b ? dense_tile_bf16_gated(tile, mode) : dense_tile_f16_gated(tile, mode);
  }
}

}  // namespace kernels
}  // namespace hipgemm

namespace {

using namespace hipgemm::detail;
namespace hk = hipgemm::kernels;

template <int kEpi>
__global__ __launch_bounds__(256) void k_dense_reduce(DenseArgs g) {
  dense_reduce_body<kEpi>(g);
}
template <int kX, bool kGated>
__global__ __launch_bounds__(256) void k_dense_slope(SlopeArgs g) {
  __shared__ float sums[8 * 256];
  dense_slope_body<kX, kGated>(g, sums);
}
__global__ __launch_bounds__(256) void k_dense_columns(const float* columns, int blocks, int N,
                                                       uint8_t* out, int type) {
  __shared__ float sums[256];
  dense_columns_body(columns, blocks, N, out, type, sums);
}

int in_bytes(int type) { return type == kInF32 ? 4 : 2; }
bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// 256 rows of an operand are addressed with 31 bits (results, dy and z with 64).
constexpr long long kMaxLd = 1 << 21;
constexpr int kMaxRows = 1 << 30;
constexpr size_t kAlign = 256;
size_t padded(size_t bytes) { return (bytes + kAlign - 1) / kAlign * kAlign; }

template <class Args>
hipError_t launch(const void* fn, dim3 grid, Args& g, hipStream_t stream) {
  if (!fn) return hipErrorInvalidValue;
  void* args[] = {&g};
  return hipLaunchKernel(fn, grid, dim3(256), args, 0, stream);
}

// ---- one product ----------------------------------------------------------------

struct Plan {
  int tile;  // index of kDenseTiles, or -1: a few rows
  int slices, slice_steps;
  long long units;
  double us;
  int first;  // columns that 256 x 256 tiles do ahead of this plan, which is for the rest
};

// Estimated times, us.  A tile's step of 64 along K by how the operands lie, and its end,
// with every CU at work on operands that come from memory: 128 x 128, 256 x 256, 64 x 128,
// 256 x 128.  Against every tile and 1, 2, 4, 8 slices on 127 shapes the choice is the best one at
// the median and within 1.5 % in the mean (us, chosen / another):
//   forward   64 x 4096 x 4096 15 (rows) / 32 (64 x 128), 64 x 14336 x 4096 29 (64 x 128 in 2
//             slices) / 46 (rows), 128 x 4096 x 14336 39 (128 x 128 in 8 slices) / 48 (in 4), 512 x
//             14336 x 4096 65 (256 x 128) / 83 (128 x 128), 1024 x 4096 x 4096 40 (128 x 128) / 55
//             (256 x 128)
//   of x      777 x 14336 x 4096 108 (256 x 128 in 2 slices) / 128 (128 x 128)
//   of w      4096 x 14336 x 4096 391 (256 x 256) / 432 (256 x 128)
struct TileTime {
  double forward, of_x, of_w, end;
};
constexpr TileTime kTime[hk::kNumDenseTiles] = {{0.57, 0.55, 0.58, 1.5},
                                                {1.55, 1.55, 1.50, 5.0},
                                                {0.40, 0.42, 0.0, 1.0},
                                                {0.85, 0.85, 0.96, 3.0}};
constexpr double kLaunch = 4.0, kSplitLaunch = 3.5;
constexpr double kBytesPerUs = 5.0e6;          // from memory: a few rows
constexpr double kSumBytesPerUs = 9.0e6;       // sums of K-slices, both ways
constexpr double kTileBytesPerUs = 5.7e6;      // the operands of tiles
constexpr double kPanelBytesPerUs = 33.5e3;    // 128 rows from memory, to the CUs that read them
constexpr double kCuBytesPerUs = 75.0e3;       // into one CU, the most of it from a cache
constexpr int kCus = 256;

double split_us(int slices, int M, int N, bool gated) {
  if (slices == 1) return 0.0;
  const double bytes = 8.0 * slices * M * (double)N * (gated ? 2 : 1);
  return kSplitLaunch + 0.3 * slices + bytes / kSumBytesPerUs;
}

// A few rows: what a CU has to fetch (x again for every 16 rows of weights), or the weights
// from memory, and more of both with more rows (gated 14336 x 4096, one row 37 us, 16 rows 51,
// 32 rows 61, 64 rows 80; tiles of 64 x 128 take 41 to 47).
double rows_us(int M, int N, int K, bool gated, int slices) {
  const int mt = M <= 16 ? 1 : M <= 32 ? 2 : 4;
  const double rows = N * (gated ? 2.0 : 1.0);
  const long long groups = (long long)((rows + 15) / 16) * slices;
  const double cu = (double)((groups + kCus - 1) / kCus) * 32.0 * (1 + mt) * K / slices;
  const double us = cu / kCuBytesPerUs, memory = 2.0 * rows * K / kBytesPerUs;
  const double more = M <= 16 ? 0.7 + 0.3 / 16 * M : 0.9 + 0.1 * mt;
  return kLaunch + (us > memory ? us : memory) * more + split_us(slices, M, N, gated);
}

// The fewest estimated us: rounds of tiles over the CUs, no less than the operands' bytes
// take, and for K-slices the way of their sums through memory.
Plan plan_whole(int kind, int M, int N, int K) {
  const int steps = (int)(((long long)K + 63) / 64);
  const bool gated = kind == hk::kDenseGated;
  const bool forward = gated || kind == hk::kDenseNT || kind == hk::kDenseRes;
  Plan best{0, 1, steps, 0, 1e300, 0};
  if (forward && M <= 64)
    for (int slices = 1; slices <= 4 && steps >= 16 * (slices - 1); slices *= 2) {
      const double us = rows_us(M, N, K, gated, slices);
      if (us < best.us) best = {-1, slices, (steps + slices - 1) / slices, 0, us, 0};
    }
  // (Of one row to four nothing else is as fast: a pass over the weights.)
  if (forward && M <= 4) return best;
  const double b_bytes = 2.0 * N * (gated ? 2.0 : 1.0) * K;
  const double whole_us = (2.0 * M * K + b_bytes) / kTileBytesPerUs;
  for (int t = 0; t < hk::kNumDenseTiles; ++t) {
    if (kind == hk::kDenseTN && t == 2) continue;
    const hk::TileShape s = hk::kDenseTiles[t];
    const int cols = gated ? s.bn / 2 : s.bn;
    const long long tiles_n = ((long long)N + cols - 1) / cols;
    const long long tiles = (((long long)M + s.bm - 1) / s.bm) * tiles_n;
    if (tiles == 0) continue;
    const double step = forward                ? kTime[t].forward
                        : kind == hk::kDenseNN ? kTime[t].of_x
                                               : kTime[t].of_w;
    for (int slices = 1; slices <= 16; ++slices) {
      if (slices > 1 && (tiles * slices > 2 * kCus || steps < 4 * slices)) break;
      const int each = (steps + slices - 1) / slices;
      const long long units = tiles * slices;
      // Where CUs stay without a tile the clock rises (1531 x 4096 x 14336, 256 x 256 in 2 slices
      // on 192 CUs: 163 us; 256 x 128 191).
      const double clock = t == 1 && units <= kCus * 3 / 4 ? 0.85 : 1.0;
      const double work =
          (double)((units + kCus - 1) / kCus) * (each * step * clock + kTime[t].end);
      // B by as many panels at once as are at work: tiles above each other share one (128 x
      // 14336 x 4096, 224 CUs: 64 x 128 39.5 us, 128 x 128 in 2 slices 34.9).
      const double panels = (double)(units < kCus ? units : kCus) * tiles_n / tiles * s.bn / 128;
      const double panels_us = b_bytes / (panels * kPanelBytesPerUs);
      const double memory = whole_us > panels_us ? whole_us : panels_us;
      const double us =
          kLaunch + (work > memory ? work : memory) + split_us(slices, M, N, gated);
      if (us < best.us) best = {t, slices, each, units, us, 0};
    }
  }
  return best;
}

// Where 256 x 256 tiles leave a last round that is not full, their whole rounds' columns by
// them and the rest as it goes best by itself, in smaller tiles or slices, in a second launch
// (us, whole / in two: 6000 x 3000 x 8192 307/253, 4096 x 5120 x 5120 213/172, gated 2048 x 14336 x
// 4096 409/373, 1531 x 14336 x 4096 170/158, 4096 x 6144 x 2048 101/96).  Two launches by estimates
// that differ by less than kGain did not differ, or were slower.
constexpr double kGain = 1.04;
Plan plan_of(int kind, int M, int N, int K) {
  Plan best = plan_whole(kind, M, N, K);
  constexpr int kBig = 1;
  const hk::TileShape s = hk::kDenseTiles[kBig];
  const int cols = kind == hk::kDenseGated ? s.bn / 2 : s.bn;
  const long long down = ((long long)M + s.bm - 1) / s.bm;
  const long long across = ((long long)N + cols - 1) / cols;
  if (best.tile < 0 || down * across <= kCus) return best;
  const double step = kind == hk::kDenseNN   ? kTime[kBig].of_x
                      : kind == hk::kDenseTN ? kTime[kBig].of_w
                                             : kTime[kBig].forward;
  const double round = ((K + 63ll) / 64) * step + kTime[kBig].end;
  const long long rounds = down * across / kCus;
  const long long first = rounds * kCus / down;  // columns of tiles
  if (first < 1 || first >= across) return best;
  const Plan rest = plan_whole(kind, M, (int)(N - first * cols), K);
  const double us = rest.us + (double)((down * first + kCus - 1) / kCus) * round;
  if (us * kGain < best.us && (rest.tile != kBig || rest.slices > 1)) {
    best = rest;
    best.us = us;
    best.first = (int)(first * cols);
  }
  return best;
}

// Columns of a partial sum's row.
long long partial_columns(int kind, int N) {
  const long long n = ((long long)N + 7) & ~7ll;
  return kind == hk::kDenseGated ? 2 * n : n;
}
size_t partial_bytes(int kind, const Plan& p, int M, int N, int parts = 1) {
  const int slices = parts * p.slices;
  if (slices == 1) return 0;
  return padded(4ull * (size_t)slices * (size_t)M * (size_t)partial_columns(kind, N - p.first));
}

// dz in parts (dense_slope_body) of so many bytes each.
struct Parts {
  int n = 1;
  long long bytes = 0;
  float scale = 1.0f;
};

hipError_t run(int x, int kind, const Plan& p, DenseArgs& g, void* ws, hipStream_t stream,
               const Parts& parts = {});

// g: operands, sizes and epilogue; ws: partial_bytes.
hipError_t product(int x, int kind, const Plan& p, DenseArgs& g, void* ws, hipStream_t stream,
                   const Parts& parts = {}) {
  if (!p.first) return run(x, kind, p, g, ws, stream, parts);
  DenseArgs part = g;
  part.N = p.first;
  const int cols = kind == hk::kDenseGated ? 128 : 256;
  const hipError_t e = run(
      x, kind,
      Plan{1, 1, 0, ((g.M + 255ll) / 256) * (p.first / cols), 0.0, 0}, part, nullptr, stream);
  if (e != hipSuccess) return e;
  const bool across = kind == hk::kDenseNN || kind == hk::kDenseTN;
  g.b += across ? 2ll * p.first : p.first * g.ldb;
  DenseEpi& o = g.epi;
  o.y += (long long)p.first * out_bytes(o.y_type);
  if (o.r) o.r += (long long)p.first * in_bytes(o.r_type);
  if (o.pre) o.pre += (long long)p.first * out_bytes(o.p_type);
  if (o.bias) o.bias += (long long)p.first * in_bytes(o.b_type);
  g.N -= p.first;
  return run(x, kind, p, g, ws, stream);
}

// With parts of A, each part's sums go to `partial` as further slices.
hipError_t run(int x, int kind, const Plan& p, DenseArgs& g, void* ws, hipStream_t stream,
               const Parts& parts) {
  const bool split = p.slices > 1 || parts.n > 1;
  g.slices = p.slices;
  g.slice_steps = p.slice_steps;
  g.partial = static_cast<float*>(ws);
  g.ldpart = partial_columns(kind, g.N);
  hipError_t e;
  if (p.tile < 0) {
    const int cols = kind == hk::kDenseGated ? 8 : 16;
    e = launch(hk::dense_rows(x, kind, g.M <= 16 ? 1 : g.M <= 32 ? 2 : 4),
               dim3((unsigned)((g.N + cols - 1) / cols), (unsigned)p.slices), g, stream);
  } else {
    const hk::TileShape s = hk::kDenseTiles[p.tile];
    const int cols = kind == hk::kDenseGated ? s.bn / 2 : s.bn;
    g.group_m = default_group_m((g.M + s.bm - 1) / s.bm, (g.N + cols - 1) / cols);
    // Weights that one row of tiles reads once go past the caches (us, with / without: 17 x 8192 x
    // 8192 29.7 / 32.5, gated 32 x 4096 x 8192 36.0 / 38.5, 64 x 8192 x 28672 117.4 / 120.5, 64 x 4096 x
    // 14336 36.5 / 37.1; nowhere slower by more than 1 %).
    const int once = s.bm == 64 && g.M <= 64 && kind != hk::kDenseNN ? hk::kDenseOnce : 0;
    const void* fn = hk::dense_tile(x, kind, p.tile, once | (split ? hk::kDenseSplit : 0));
    const dim3 grid((unsigned)(p.units < kCus ? p.units : kCus));
    e = launch(fn, grid, g, stream);
    for (int n = 1; n < parts.n && e == hipSuccess; ++n) {
      g.a += parts.bytes;
      g.partial += (long long)p.slices * g.M * g.ldpart;
      e = launch(fn, grid, g, stream);
    }
    g.partial = static_cast<float*>(ws);
  }
  if (e != hipSuccess || !split) return e;
  if (parts.n > 1) {
    g.part_slices = p.slices;
    g.part_scale = parts.scale;
    g.slices = parts.n * p.slices;
  }
  const long long threads = (long long)g.M * ((g.N + 7) / 8);
  const void* fn = kind == hk::kDenseGated ? (const void*)&k_dense_reduce<kEpiGated>
                   : kind == hk::kDenseRes ? (const void*)&k_dense_reduce<kEpiResidual>
                   : kind == hk::kDenseNT  ? (const void*)&k_dense_reduce<kEpiLinear>
                                           : (const void*)&k_dense_reduce<kEpiPlain>;
  return launch(fn, dim3((unsigned)((threads + 255) / 256)), g, stream);
}

bool operand(const void* p, long long ld, long long columns) {
  return p && aligned(p, 16) && ld >= columns && ld % 8 == 0 && ld <= kMaxLd;
}
bool result(const void* p, long long ld, long long columns, int out) {
  return p && aligned(p, (uintptr_t)out_bytes(out)) && ld >= columns;
}

bool common(int M, int N, int K, int gated, int type, int act) {
  return M >= 0 && M <= kMaxRows && N >= 0 && K >= 0 && K % 8 == 0 && (gated == 0 || gated == 1) &&
         (!gated || N % 8 == 0) && (long long)N * (gated ? 2 : 1) <= kMaxLd && K <= kMaxLd &&
         (type == HIPGEMM_IN_BF16 || type == HIPGEMM_IN_F16) && act >= 0 &&
         act <= HIPGEMM_ACT_SILU;
}

// ---- forward ----------------------------------------------------------------------

hipError_t check(const hipgemm_linear_desc* desc) {
  if (!desc || desc->size != sizeof(hipgemm_linear_desc)) return hipErrorInvalidValue;
  const hipgemm_linear_desc& d = *desc;
  if (!common(d.M, d.N, d.K, d.gated, d.type, d.activation) || d.out_dtype < 0 ||
      d.out_dtype > HIPGEMM_OUT_F32 || d.bias_type < 0 || d.bias_type > HIPGEMM_IN_F16 ||
      d.residual_type < 0 || d.residual_type > HIPGEMM_IN_F16 || d.pre_dtype < 0 ||
      d.pre_dtype > HIPGEMM_OUT_F32 || (d.gated && d.residual))
    return hipErrorInvalidValue;
  if (d.M == 0 || d.N == 0) return hipSuccess;
  const long long rows = d.gated ? 2ll * d.N : d.N;
  if (!result(d.y, d.ldy, d.N, d.out_dtype) ||
      (d.K > 0 && (!operand(d.x, d.ldx, d.K) || !operand(d.weight, d.ldw, d.K))) ||
      (d.bias && !aligned(d.bias, in_bytes(d.bias_type))) ||
      (d.residual && (!aligned(d.residual, in_bytes(d.residual_type)) || d.ldr < d.N)) ||
      (d.pre && !result(d.pre, d.ldp, rows, d.pre_dtype)))
    return hipErrorInvalidValue;
  return hipSuccess;
}

int kind_of(const hipgemm_linear_desc& d) {
  return d.gated ? hk::kDenseGated : d.residual ? hk::kDenseRes : hk::kDenseNT;
}

size_t forward_bytes(const hipgemm_linear_desc& d) {
  const int kind = kind_of(d);
  return partial_bytes(kind, plan_of(kind, d.M, d.N, d.K), d.M, d.N);
}

hipError_t forward(const hipgemm_linear_desc& d, hipStream_t stream) {
  const int kind = kind_of(d);
  const Plan p = plan_of(kind, d.M, d.N, d.K);
  const size_t need = partial_bytes(kind, p, d.M, d.N);
  if (need && (!d.workspace || d.workspace_bytes < need || !aligned(d.workspace, kAlign)))
    return hipErrorInvalidValue;
  DenseArgs g{};
  g.a = static_cast<const uint8_t*>(d.x);
  g.b = static_cast<const uint8_t*>(d.weight);
  // Strides of operands without elements may be anything and are not looked at: ranges of
  // buffers are made of them, which have to be empty.
  if (d.K > 0) {
    g.lda = 2 * d.ldx;
    g.ldb = 2 * d.ldw;
    g.up = 2 * d.ldw * d.N;
  }
  g.M = d.M;
  g.N = d.N;
  g.K = d.K;
  DenseEpi& e = g.epi;
  e.y = static_cast<uint8_t*>(d.y);
  e.bias = static_cast<const uint8_t*>(d.bias);
  e.r = static_cast<const uint8_t*>(d.residual);
  e.pre = static_cast<uint8_t*>(d.pre);
  e.ldy = d.ldy;
  e.ldr = d.ldr;
  e.ldp = d.ldp;
  e.up = d.N;
  e.act = d.activation;
  e.y_type = d.out_dtype;
  e.p_type = d.pre_dtype;
  e.b_type = d.bias_type;
  e.r_type = d.residual_type;
  return product(d.type, kind, p, g, d.workspace, stream);
}

// ---- backward ---------------------------------------------------------------------

hipError_t check(const hipgemm_linear_grad_desc* desc) {
  if (!desc || desc->size != sizeof(hipgemm_linear_grad_desc)) return hipErrorInvalidValue;
  const hipgemm_linear_grad_desc& d = *desc;
  if (!common(d.M, d.N, d.K, d.gated, d.type, d.activation) || d.dy_type < 0 ||
      d.dy_type > HIPGEMM_IN_F16 || d.pre_type < 0 || d.pre_type > HIPGEMM_IN_F16 ||
      d.dx_dtype < 0 || d.dx_dtype > HIPGEMM_OUT_F32 || d.dw_dtype < 0 ||
      d.dw_dtype > HIPGEMM_OUT_F32 || d.db_dtype < 0 || d.db_dtype > HIPGEMM_OUT_F32)
    return hipErrorInvalidValue;
  const long long cols = d.gated ? 2ll * d.N : d.N;
  if (d.M > 0 && d.N > 0) {
    if (!d.dy || !aligned(d.dy, in_bytes(d.dy_type)) || d.lddy < d.N) return hipErrorInvalidValue;
    if ((d.gated || d.activation != HIPGEMM_ACT_NONE) &&
        (!d.pre || !aligned(d.pre, in_bytes(d.pre_type)) || d.ldp < cols))
      return hipErrorInvalidValue;
    if (d.K > 0 && ((d.dx && !operand(d.weight, d.ldw, d.K)) ||
                    (d.dw && !operand(d.x, d.ldx, d.K))))
      return hipErrorInvalidValue;
  }
  if ((d.dx && !result(d.dx, d.lddx, d.K, d.dx_dtype)) ||
      (d.dw && !result(d.dw, d.lddw, d.K, d.dw_dtype)) ||
      (d.db && !aligned(d.db, (uintptr_t)out_bytes(d.db_dtype))))
    return hipErrorInvalidValue;
  return hipSuccess;
}

// Where dz is dy itself: nothing to multiply by, in the operands' type, in rows that the
// products read as they are.
bool as_is(const hipgemm_linear_grad_desc& d) {
  return !d.gated && d.activation == HIPGEMM_ACT_NONE && d.dy_type == d.type && d.N % 8 == 0 &&
         aligned(d.dy, 16) && d.lddy % 8 == 0 && d.lddy <= kMaxLd;
}

struct GradPlan {
  long long cols, ldz;  // of dz
  bool own;             // dz lies in the workspace
  int blocks, rows;     // of the column sums
  int parts_x, parts_w; // of dz, that dx and dw are sums over
  long long plane;      // elements of a part
  size_t dz, columns, partial;
  Plan of_x, of_w;
  bool together;        // of_x and of_w in one launch
};

// Both products in tiles of 128 x 128 that have a CU each, or one after the other: by sizes
// alone, so that a gradient is the same with and without the others, and where neither alone
// takes more than kAlone times its best by the estimates (bf16, with dz, us: both / the slowed one
// alone, one after the other and together;  of dx at 1.22 times its best, 1531 x 2001 x 1000:
// 42.8, 32.2 / 25.1, 31.8;  gated 1.19, 2048 x 704 x 1024: 38.4, 30.0 / 20.7, 23.9;  of dw at 1.44,
// 2048 x 512 x 1024: 24.2, 19.8 / 16.8, 19.2;  past it, of dx gated at 1.56, 777 x 1400 x 1000: 39.8,
// 37.3 / 25.8, 36.3;  1.84, 1024 x 1408 x 512: 35.5, 32.9 / 23.2, 32.5).
constexpr double kAlone = 1.5;
void pair_plan(const hipgemm_linear_grad_desc& d, GradPlan& p) {
  p.of_x = plan_of(hk::kDenseNN, d.M, d.K, (int)p.cols);
  p.of_w = plan_of(hk::kDenseTN, (int)p.cols, d.K, d.M);
  const hk::TileShape s = hk::kDenseTiles[0];
  const long long across = ((long long)d.K + s.bn - 1) / s.bn;
  const long long x = (((long long)d.M + s.bm - 1) / s.bm) * across;
  const long long w = ((p.cols + s.bm - 1) / s.bm) * across;
  const int steps_x = (int)((p.cols + 63) / 64), steps_w = (int)(((long long)d.M + 63) / 64);
  const double of_x = kLaunch + steps_x * kTime[0].of_x + kTime[0].end;
  const double of_w = kLaunch + steps_w * kTime[0].of_w + kTime[0].end;
  const double us = of_x > of_w ? of_x : of_w;
  p.together = x > 0 && w > 0 && x + w <= kCus && us < p.of_x.us + p.of_w.us &&
               of_x <= kAlone * p.of_x.us && of_w <= kAlone * p.of_w.us;
  if (p.together) {
    p.of_x = {0, 1, steps_x, x, us, 0};
    p.of_w = {0, 1, steps_w, w, us, 0};
  }
  // (Sums over parts go through memory: no columns apart, no launch with another product.)
  if (p.parts_x > 1) p.of_x = plan_whole(hk::kDenseNN, d.M, d.K, (int)p.cols);
  if (p.parts_w > 1) p.of_w = plan_whole(hk::kDenseTN, (int)p.cols, d.K, d.M);
  if (p.parts_x > 1 || p.parts_w > 1) p.together = false;
}
GradPlan grad_plan(const hipgemm_linear_grad_desc& d) {
  GradPlan p{};
  p.cols = d.gated ? 2ll * d.N : d.N;
  p.ldz = (p.cols + 7) & ~7ll;
  p.own = !as_is(d) && (d.dx || d.dw);
  // Blocks of kSlopeColumns columns by `rows` rows: 32 to a CU, of eight rows at least (us,
  // 4 / 16 / 32 to a CU: 4096 x 16384 with fp32 sums 137 / 131 / 125 = 4.3 TB/s, gated 4096 x 14336
  // 190 / 169 / 164 = 5.0 TB/s).
  const int across = (d.N + kSlopeColumns - 1) / kSlopeColumns;
  int blocks = across ? (32 * kCus + across - 1) / across : 1;
  if (blocks > (d.M + 7) / 8) blocks = (d.M + 7) / 8;
  if (blocks < 1) blocks = 1;
  p.rows = ((d.M + blocks - 1) / blocks + 7) / 8 * 8;
  if (p.rows < 8) p.rows = 8;
  p.blocks = (d.M + p.rows - 1) / p.rows;
  if (p.blocks < 1) p.blocks = 1;
  const int parts = d.type == HIPGEMM_IN_BF16 ? 3 : 2;
  p.parts_x = !as_is(d) && d.dx && d.dx_dtype == HIPGEMM_OUT_F32 ? parts : 1;
  p.parts_w = !as_is(d) && d.dw && d.dw_dtype == HIPGEMM_OUT_F32 ? parts : 1;
  const size_t plane = padded(2ull * (size_t)d.M * (size_t)p.ldz);
  p.plane = (long long)(plane / 2);
  p.dz = p.own ? plane * (size_t)(p.parts_x > p.parts_w ? p.parts_x : p.parts_w) : 0;
  p.columns = d.db ? padded(4ull * (size_t)p.blocks * (size_t)p.cols) : 0;
  pair_plan(d, p);
  size_t part = 0;
  if (d.dx) part = partial_bytes(hk::kDenseNN, p.of_x, d.M, d.K, p.parts_x);
  if (d.dw) {
    const size_t w = partial_bytes(hk::kDenseTN, p.of_w, (int)p.cols, d.K, p.parts_w);
    if (w > part) part = w;
  }
  p.partial = part;
  return p;
}

void plain_epilogue(DenseArgs& g, void* y, long long ldy, int out) {
  g.epi.y = static_cast<uint8_t*>(y);
  g.epi.ldy = ldy;
  g.epi.y_type = out;
}

hipError_t backward(const hipgemm_linear_grad_desc& d, hipStream_t stream) {
  const GradPlan p = grad_plan(d);
  const size_t need = p.dz + p.columns + p.partial;
  if (need && (!d.workspace || d.workspace_bytes < need || !aligned(d.workspace, kAlign)))
    return hipErrorInvalidValue;
  uint8_t* ws = static_cast<uint8_t*>(d.workspace);
  uint8_t* dz = ws;
  float* columns = reinterpret_cast<float*>(ws + p.dz);
  void* partial = ws + p.dz + p.columns;
  if (p.own || d.db) {
    SlopeArgs s{};
    s.dy = static_cast<const uint8_t*>(d.dy);
    s.pre = d.activation == HIPGEMM_ACT_NONE && !d.gated ? nullptr
                                                         : static_cast<const uint8_t*>(d.pre);
    s.dz = p.own ? dz : nullptr;
    s.columns = d.db ? columns : nullptr;
    s.lddy = d.lddy;
    s.ldp = d.ldp;
    s.lddz = p.ldz;
    s.M = d.M;
    s.N = d.N;
    s.act = d.activation;
    s.dy_type = d.dy_type;
    s.p_type = d.pre_type;
    s.rows = p.rows;
    s.parts = p.parts_x > p.parts_w ? p.parts_x : p.parts_w;
    s.plane = p.plane;
    const dim3 grid((unsigned)((d.N + kSlopeColumns - 1) / kSlopeColumns), (unsigned)p.blocks);
    const bool b = d.type == HIPGEMM_IN_BF16;
    const void* fn = d.gated ? (b ? (const void*)&k_dense_slope<kInBf16, true>
                                  : (const void*)&k_dense_slope<kInF16, true>)
                             : (b ? (const void*)&k_dense_slope<kInBf16, false>
                                  : (const void*)&k_dense_slope<kInF16, false>);
    if (d.N > 0) {
      const hipError_t e = launch(fn, grid, s, stream);
      if (e != hipSuccess) return e;
      if (d.db) {
        int blocks = p.blocks, cols = (int)p.cols, type = d.db_dtype;
        uint8_t* out = static_cast<uint8_t*>(d.db);
        const float* from = columns;
        void* args[] = {&from, &blocks, &cols, &out, &type};
        const hipError_t e2 =
            hipLaunchKernel((const void*)&k_dense_columns, dim3((unsigned)((cols + 15) / 16)),
                            dim3(256), args, 0, stream);
        if (e2 != hipSuccess) return e2;
      }
    }
  }
  const uint8_t* z = p.own ? dz : static_cast<const uint8_t*>(d.dy);
  const long long ldz = p.own ? p.ldz : d.lddy;
  const bool of_x = d.dx && d.M > 0 && d.K > 0, of_w = d.dw && d.N > 0 && d.K > 0;
  DenseArgs x{}, w{};
  x.a = w.a = z;
  if (d.M > 0 && d.N > 0) x.lda = w.lda = 2 * ldz;  // (as in forward)
  x.b = static_cast<const uint8_t*>(d.weight);
  if (d.N > 0) x.ldb = 2 * d.ldw;
  w.b = static_cast<const uint8_t*>(d.x);
  if (d.M > 0) w.ldb = 2 * d.ldx;
  x.M = w.K = d.M;
  x.K = w.M = (int)p.cols;
  x.N = w.N = d.K;
  plain_epilogue(x, d.dx, d.lddx, d.dx_dtype);
  plain_epilogue(w, d.dw, d.lddw, d.dw_dtype);
  if (of_x && of_w && p.together) {
    const hk::TileShape s = hk::kDenseTiles[0];
    const int across = (d.K + s.bn - 1) / s.bn;
    x.slices = w.slices = 1;
    x.group_m = default_group_m((x.M + s.bm - 1) / s.bm, across);
    w.group_m = default_group_m((w.M + s.bm - 1) / s.bm, across);
    DensePair pair{x, w, (int)p.of_x.units};
    return launch(hk::dense_pair(d.type), dim3((unsigned)(p.of_x.units + p.of_w.units)), pair,
                  stream);
  }
  const float scale = d.type == HIPGEMM_IN_BF16 ? 1.0f / kRest<kInBf16> : 1.0f / kRest<kInF16>;
  if (of_x) {
    const hipError_t e = product(d.type, hk::kDenseNN, p.of_x, x, partial, stream,
                                 Parts{p.parts_x, 2 * p.plane, scale});
    if (e != hipSuccess) return e;
  }
  return of_w ? product(d.type, hk::kDenseTN, p.of_w, w, partial, stream,
                        Parts{p.parts_w, 2 * p.plane, scale})
              : hipSuccess;
}

hipgemm_linear_plan shown(const Plan& p) {
  if (p.tile < 0) return {0, 0, p.slices, p.first};
  return {hk::kDenseTiles[p.tile].bm, hk::kDenseTiles[p.tile].bn, p.slices, p.first};
}

}  // namespace

extern "C" size_t hipgemm_linear_workspace_size(const hipgemm_linear_desc* desc) {
  if (!desc || desc->size != sizeof(*desc) ||
      !common(desc->M, desc->N, desc->K, desc->gated, desc->type, desc->activation) ||
      desc->M == 0 || desc->N == 0)
    return 0;
  return forward_bytes(*desc);
}

extern "C" hipError_t hipgemm_linear(const hipgemm_linear_desc* desc, hipStream_t stream) {
  const hipError_t e = check(desc);
  return e != hipSuccess || desc->M == 0 || desc->N == 0 ? e : forward(*desc, stream);
}

extern "C" size_t hipgemm_linear_backward_workspace_size(const hipgemm_linear_grad_desc* desc) {
  if (!desc || desc->size != sizeof(*desc) ||
      !common(desc->M, desc->N, desc->K, desc->gated, desc->type, desc->activation))
    return 0;
  const GradPlan p = grad_plan(*desc);
  return p.dz + p.columns + p.partial;
}

extern "C" hipError_t hipgemm_linear_backward(const hipgemm_linear_grad_desc* desc,
                                              hipStream_t stream) {
  const hipError_t e = check(desc);
  return e != hipSuccess ? e : backward(*desc, stream);
}

extern "C" hipError_t hipgemm_linear_select(const hipgemm_linear_desc* desc,
                                            hipgemm_linear_plan* plan) {
  if (!plan || !desc || desc->size != sizeof(*desc) ||
      !common(desc->M, desc->N, desc->K, desc->gated, desc->type, desc->activation))
    return hipErrorInvalidValue;
  *plan = {};
  if (desc->M > 0 && desc->N > 0)
    *plan = shown(plan_of(kind_of(*desc), desc->M, desc->N, desc->K));
  return hipSuccess;
}

extern "C" hipError_t hipgemm_linear_backward_select(const hipgemm_linear_grad_desc* desc,
                                                     hipgemm_linear_plan plan[2]) {
  if (!plan || !desc || desc->size != sizeof(*desc) ||
      !common(desc->M, desc->N, desc->K, desc->gated, desc->type, desc->activation))
    return hipErrorInvalidValue;
  const GradPlan p = grad_plan(*desc);
  plan[0] = plan[1] = {};
  if (desc->dx && desc->M > 0 && desc->K > 0) plan[0] = shown(p.of_x);
  if (desc->dw && desc->N > 0 && desc->K > 0) plan[1] = shown(p.of_w);
  return hipSuccess;
}
