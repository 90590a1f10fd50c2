// hipgemm_moe_experts: arguments and launches.
#include "hipgemm.h"

#include <cmath>

#include "kernels.hpp"

#include "hipgemm/detail/moe_vec.hpp"

namespace hipgemm {
namespace kernels {

#define HIPGEMM_MOE(W)                                  \
  const void* moe_up_bf16_##W(int s, int mode, int mt, int wk); \
  const void* moe_up_f16_##W(int s, int mode, int mt, int wk);  \
  const void* moe_down_##W(int s, int mode, int mt, int wk, int h); \
  const void* moe_vec_up_bf16_##W(int s, int lk);       \
  const void* moe_vec_up_f16_##W(int s, int lk);        \
  const void* moe_vec_down_##W(int s, int lk, int h);
HIPGEMM_MOE(int4)
HIPGEMM_MOE(int4z)
HIPGEMM_MOE(fp4)
HIPGEMM_MOE(e4m3)
#undef HIPGEMM_MOE

const void* moe_up(int x, int w, int s, int mode, int mt, int wk) {
  const bool b = x == detail::kInBf16;
  switch (w) {
    case detail::kWInt4: return b ? moe_up_bf16_int4(s, mode, mt, wk) : moe_up_f16_int4(s, mode, mt, wk);
    case detail::kWInt4Z:
      return b ? moe_up_bf16_int4z(s, mode, mt, wk) : moe_up_f16_int4z(s, mode, mt, wk);
    case detail::kWFp4: return b ? moe_up_bf16_fp4(s, mode, mt, wk) : moe_up_f16_fp4(s, mode, mt, wk);
    default: return b ? moe_up_bf16_e4m3(s, mode, mt, wk) : moe_up_f16_e4m3(s, mode, mt, wk);
  }
}
const void* moe_down(int w, int s, int mode, int mt, int wk, int h) {
  switch (w) {
    case detail::kWInt4: return moe_down_int4(s, mode, mt, wk, h);
    case detail::kWInt4Z: return moe_down_int4z(s, mode, mt, wk, h);
    case detail::kWFp4: return moe_down_fp4(s, mode, mt, wk, h);
    default: return moe_down_e4m3(s, mode, mt, wk, h);
  }
}
const void* moe_vec_up(int x, int w, int s, int lk) {
  const bool b = x == detail::kInBf16;
  switch (w) {
    case detail::kWInt4: return b ? moe_vec_up_bf16_int4(s, lk) : moe_vec_up_f16_int4(s, lk);
    case detail::kWInt4Z: return b ? moe_vec_up_bf16_int4z(s, lk) : moe_vec_up_f16_int4z(s, lk);
    case detail::kWFp4: return b ? moe_vec_up_bf16_fp4(s, lk) : moe_vec_up_f16_fp4(s, lk);
    default: return b ? moe_vec_up_bf16_e4m3(s, lk) : moe_vec_up_f16_e4m3(s, lk);
  }
}
const void* moe_vec_down(int w, int s, int lk, int h) {
  switch (w) {
    case detail::kWInt4: return moe_vec_down_int4(s, lk, h);
    case detail::kWInt4Z: return moe_vec_down_int4z(s, lk, h);
    case detail::kWFp4: return moe_vec_down_fp4(s, lk, h);
    default: return moe_vec_down_e4m3(s, lk, h);
  }
}

}  // namespace kernels
}  // namespace hipgemm

namespace {

using namespace hipgemm::detail;
namespace hk = hipgemm::kernels;

static_assert(HIPGEMM_W8_E4M3 == kWE4M3 && HIPGEMM_MOE_MAX_PAIRS == kMoePairs &&
                  HIPGEMM_MOE_MAX_EXPERTS == kMoeExperts, "codes");

// Four columns of one token per thread, eight pairs' loads at a time.
__global__ __launch_bounds__(256) void k_moe_sum(MoeArgs g) {
  const int i = (int)blockIdx.x * 256 + (int)threadIdx.x, per = g.D / 4;
  const int t = i / per, d = i % per * 4;
  if (t >= g.T) return;
  const long long pairs = g.T * g.k;
  f32x4 v = {};
  for (int j0 = 0; j0 < g.k; j0 += 8) {
    bool on[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = g.ids[t * g.k + min(j0 + j, g.k - 1)];
      on[j] = j0 + j < g.k && e >= 0 && e < g.E;
    }
    for (int q = 0; q < g.parts; ++q) {
      f32x4 o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        o[j] = *reinterpret_cast<const f32x4*>(
            g.o + (q * pairs + t * g.k + min(j0 + j, g.k - 1)) * g.D + d);
      // (what was not written may be anything)
#pragma unroll
      for (int j = 0; j < 8; ++j) v = on[j] ? v + o[j] : v;
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) store_result(g.y, t * g.ldy + d + c, g.out, v[c]);
}

bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

constexpr int kMaxDim = 1 << 26;           // Stream's group index
constexpr long long kMaxRow = 1 << 25;  // 32 rows in a buffer's range

// Tokens of one turn.
int turn_tokens(int T, int k) { return T < kMoePairs / k ? T : kMoePairs / k; }

int mode_of(int x_type, int format, int scale_type, int group) {
  if (format == kWE4M3) return kNone;
  if (format == kWFp4 && scale_type == kScaleE8M0 && x_type == kInBf16) return kInline;
  return group % 128 == 0 ? kCoarse : kFine;
}

bool matrix_ok(const hipgemm_moe_matrix& m, int rows, int K, const hipgemm_moe_desc& d) {
  const bool e4m3 = d.format == HIPGEMM_W8_E4M3;
  const long long row = e4m3 ? K : K / 2;
  const long long groups = e4m3 ? 1 : (K - 1) / d.group_size + 1;
  return m.weight && m.scales && aligned(m.weight, 16) && m.ldw <= kMaxRow &&
         m.lds <= kMaxRow / type_bytes(d.scale_type) &&
         aligned(m.scales, type_bytes(d.scale_type)) && m.ldw >= row && m.ldw % 16 == 0 &&
         m.expert_w % 16 == 0 && (d.E == 1 || m.expert_w >= (rows - 1) * m.ldw + row) &&
         m.lds >= groups && (d.E == 1 || m.expert_s >= (rows - 1) * m.lds + groups) &&
         (!m.zeros || d.format == HIPGEMM_W4_INT4);
}

// Experts that are chosen, if all are chosen alike.
double chosen_experts(int T, int k, int E) {
  return E * (1.0 - std::pow(1.0 - (k < E ? (double)k / E : 1.0), T));
}

// What a workgroup of the grouped kernels keeps in LDS is the same for all formats.
template <int kMT, int kParts>
using AnyStream = Stream<kInBf16, kWE4M3, kInF32, kNone, kMT, kParts, 8, kMoeTables>;
// Rows of x (of D elements) going up.
int up_rows(int mt, int D) {
  return mt == 2 ? AnyStream<2, 1>::rows_that_fit(D) : AnyStream<1, 1>::rows_that_fit(D);
}
// Parts of h (moe.hpp).
int h_parts(int out_dtype) { return out_dtype == HIPGEMM_OUT_F32 ? 3 : 2; }
// Elements of h going down, over all rows.
int down_elems(int mt, int h) {
  return h == 3 ? AnyStream<1, 3>::kElems / 3
                : (mt == 2 ? AnyStream<2, 2>::kElems : AnyStream<1, 2>::kElems) / 2;
}

// Whether the grouped kernels take the sizes: a row of x in LDS going up, and going
// down no more parts than 64.
bool grouped(int D, int F) { return up_rows(1, D) >= 1 && F <= 1 << 16; }

// The down product: tiles of 16 rows of h per group, and parts of F, of len (a
// multiple of 256).
struct DownPlan {
  int mt, parts, len;
};
DownPlan down_plan(int T, int k, int E, int D, int F, int h) {
  const int pairs = T * k, steps = (F + 255) / 256;
  // Parts so short that the rows of an expert, up to half as many again as there are on
  // average, lie in LDS together: its weights are read once for them.  Not below
  // 1024, and of 32 rows only where more than 16 fit.
  const double rows = std::ceil(1.5 * pairs / chosen_experts(T, k, E));
  int mt = pairs > 12 * E && h == 2 ? 2 : 1, fit;
  for (;; mt = 1) {
    fit = (int)(down_elems(mt, h) / (rows < 16 * mt ? rows : 16 * mt)) / 256;
    if (fit < 4) fit = 4;
    if (mt == 1 || down_elems(2, h) / (256 * (fit < steps ? fit : steps)) > 16) break;
  }
  const int chosen = pairs < E ? pairs : E;  // experts at most
  const int tiles = chosen * ((D + 63) / 64);
  int parts = tiles >= 512 ? 1 : (512 + tiles - 1) / tiles;
  if (parts > (steps + 7) / 8) parts = (steps + 7) / 8;
  if (parts < (steps + fit - 1) / fit) parts = (steps + fit - 1) / fit;
  const int len = (steps + parts - 1) / parts;
  return {mt, (steps + len - 1) / len, 256 * len};
}

hipError_t launch(const void* fn, dim3 grid, int threads, MoeArgs& g, hipStream_t stream) {
  if (!fn) return hipErrorInvalidValue;
  void* args[] = {&g};
  return hipLaunchKernel(fn, grid, dim3((unsigned)threads), args, 0, stream);
}

// Lanes of a row for rows of K elements (16 bytes of weights a lane): 16 where 64
// would leave most of them idle.
int vec_lanes(int K, int per_lane) { return K / per_lane > 24 ? 64 : 16; }
int chunks_of(int K, int per_lane, int lk) {
  return (K + per_lane * lk - 1) / (per_lane * lk);
}

hipError_t vec_turn(MoeArgs g, const hipgemm_moe_desc& d, hipStream_t stream) {
  const int per_lane = d.format == HIPGEMM_W8_E4M3 ? 16 : 32;
  auto steps_of = [](int rows, int groups, int step) {  // of a wave: 512 workgroups
    const int s = (rows + 512 * step / groups - 1) / (512 * step / groups > 0 ? 512 * step / groups : 1);
    const int most = kVecMaxRows / step;
    return s < 1 ? 1 : s > most ? most : s;
  };
  {
    const int lk = vec_lanes(g.D, per_lane), chunks = chunks_of(g.D, per_lane, lk);
    const int step = kVecRows * (kWave / lk), turns = (chunks + 3) / 4;
    g.waves_k = (chunks + turns - 1) / turns;
    const int waves_r = g.waves_k > 2 ? 1 : 4 / g.waves_k;  // pairs of gate and up
    g.wave_rows = step * steps_of((g.F + waves_r - 1) / waves_r, g.T * g.k, step);
    g.rows = g.wave_rows * waves_r;
    if (g.rows > kVecMaxRows * waves_r) return hipErrorInvalidValue;
    const hipError_t e = launch(
        hk::moe_vec_up(d.x_type, d.w13.zeros ? kWInt4Z : d.format, d.scale_type, lk),
        dim3((unsigned)((g.F + g.rows - 1) / g.rows), (unsigned)(g.T * g.k)),
        kWave * g.waves_k * 2 * waves_r, g, stream);
    if (e != hipSuccess) return e;
  }
  const int lk = vec_lanes(g.F, per_lane), chunks = chunks_of(g.F, per_lane, lk);
  const int items = chunks * g.k, turns = (items + 7) / 8;
  g.rows = kVecRows * (kWave / lk) * steps_of(g.D, g.T, kVecRows * (kWave / lk));
  return launch(hk::moe_vec_down(d.w2.zeros ? kWInt4Z : d.format, d.scale_type, lk, g.h_parts),
                dim3((unsigned)((g.D + g.rows - 1) / g.rows), (unsigned)g.T),
                kWave * ((items + turns - 1) / turns), g, stream);
}

// The kernels of a turn.
hipgemm_moe_plan turn_plan(int T, int k, int E, int D, int F, int format, int h) {
  const int pairs = T * k;
  const double chosen = chosen_experts(T, k, E);
  // Pair by pair while few experts are read twice.  us in a graph, pairs / grouped,
  // by tokens, ids spread evenly: int4, 8 of 64 experts of 2048 x 1024, 2 24/29, 12
  // 86/62; 8 of 128 of 4096 x 1536, 4 71/81, 8 120/119, 16 223/175;  fp4, 3 of 30 of 2336
  // x 1056, 5 25/40;  e4m3, 4 of 64 of 4096 x 2048, 2 41/51, 4 71/80, 8 127/115; 2 of 8
  // of 4096 x 14336, 1 69/72, 2 121/115.  (Grouped, 4-bit weights stream at 3 to 4.6
  // TB/s, e4m3 ones at 5 to 5.8.)
  // And while what is read again is less than 64 MB: grouping is a third launch and
  // the tables.  Pairs / grouped, MB: e4m3 10 tokens, 1 of 24 of 384 x 640, 1, 9.5/20;
  // 2, 7 of 24 of 768 x 1536, 7, 18.7/29;  int4 3, 3 of 4 of 1536 x 384, 4, 12/24;  64, 2
  // of 4 of 256 x 512, 24, 16/29;  6, 8 of 64 of 2048 x 1024, 40, 54/51;  e4m3 64, 4 of 8
  // of 256 x 256, 49, 12.5/33;  fp4 12, 3 of 30 of 2336 x 1056, 54, 44/53;  32, 4 of 64 of
  // 1024 x 512, 57, 30/36;  e4m3 41, 1 of 16 of 1024 x 896, 72, 29/26;  int4 64, 8 of 128
  // of 512 x 512, 152, 50/38.  Decided wrongly: fp4 10, 5 of 16 of 4096 x 256, 54, 34/28.
  const bool e4m3 = format == HIPGEMM_W8_E4M3;
  const double expert_bytes = 3.0 * D * F * (e4m3 ? 1.0 : 0.5);
  if (!grouped(D, F) || pairs <= chosen * (e4m3 ? 1.13 : 1.5) ||
      (pairs - chosen) * expert_bytes <= 64e6)
    return {};
  // Tiles of 16 tokens, two at a time where experts have more on average and more
  // rows than with one fit in LDS (sums of two tiles take room from them).
  const int mt = pairs > 12 * E && up_rows(2, D) > up_rows(1, D) ? 2 : 1;
  const DownPlan down = down_plan(T, k, E, D, F, h);
  // Tiles of 128 rows with two waves to a row's K where each CU has ten or more of
  // them (fewer ends of tiles per byte), of 32 rows with eight where not, unless K is
  // no more than one unit for each of the eight: most would wait (us, eight / two:
  // fp4 320 x 6272, 6 of 12, 26 tokens 73/51;  int4 2048 x 1024, 8 of 64, 64 tokens
  // 85/64;  e4m3 1024 x 512, 8 of 128, 64 tokens 64/53;  beyond, e4m3 4096 x 4096, 2 of
  // 8, 16 tokens 82/91, 4096 x 2048, 4 of 64, 177/187).
  const int short_k = 8 * (e4m3 ? 128 : 256);
  const int wku = chosen * F / 64 >= 2560 || D <= short_k ? 2 : 8;
  const int wkd = chosen * D / 128 * down.parts >= 2560 || down.len <= short_k ? 2 : 8;
  return {1, 16 * mt, wku, 16 * down.mt, wkd, down.parts, down.len};
}

hipError_t turn(MoeArgs g, const hipgemm_moe_desc& d, hipStream_t stream) {
  const hipgemm_moe_plan p = turn_plan(g.T, g.k, g.E, g.D, g.F, d.format, g.h_parts);
  if (!p.grouped) return vec_turn(g, d, stream);
  g.parts = p.parts;
  g.part_len = p.part_len;
  const int cus = 256;
  hipError_t e = launch(hk::moe_up(d.x_type, d.w13.zeros ? kWInt4Z : d.format, d.scale_type,
                                   mode_of(d.x_type, d.format, d.scale_type, d.group_size),
                                   p.up_rows / 16, p.up_waves),
                        dim3((unsigned)cus), 512, g, stream);
  if (e != hipSuccess) return e;
  e = launch(hk::moe_down(d.w2.zeros ? kWInt4Z : d.format, d.scale_type,
                          mode_of(kInBf16, d.format, d.scale_type, d.group_size), p.down_rows / 16,
                          p.down_waves, g.h_parts),
             dim3((unsigned)cus), 512, g, stream);
  if (e != hipSuccess) return e;
  return launch((const void*)&k_moe_sum, dim3((unsigned)((g.T * (g.D / 4) + 255) / 256)), 256, g,
                stream);
}

}  // namespace

extern "C" hipError_t hipgemm_moe_select(int T, int k, int E, int D, int F, int format,
                                         int out_dtype, hipgemm_moe_plan* plan) {
  if (!plan || T < 1 || k < 1 || k > 64 || E < 1 || E > HIPGEMM_MOE_MAX_EXPERTS || D < 32 ||
      D % 32 != 0 || D > kMaxDim || F < 32 || F % 32 != 0 || F > kMaxDim / 2 || format < 0 ||
      format > HIPGEMM_W8_E4M3 || out_dtype < 0 || out_dtype > HIPGEMM_OUT_F32)
    return hipErrorInvalidValue;
  *plan = turn_plan(turn_tokens(T, k), k, E, D, F, format, h_parts(out_dtype));
  return hipSuccess;
}

extern "C" size_t hipgemm_moe_workspace_size(int T, int k, int E, int D, int F) {
  if (T <= 0 || k <= 0 || k > 64 || E <= 0 || D <= 0 || F <= 0) return 0;
  const int t = turn_tokens(T, k);
  // (a last turn of fewer tokens can have more parts, and h of three parts)
  size_t o = 0;
  for (int u : {t, T % t})
    for (int h : {2, 3}) {
      if (u == 0 || !grouped(D, F)) continue;
      const size_t n = (size_t)down_plan(u, k, E, D, F, h).parts * u * k;
      if (n > o) o = n;
    }
  return (size_t)t * k * F * 6 + o * D * 4;
}

extern "C" hipError_t hipgemm_moe_experts(const hipgemm_moe_desc* desc, hipStream_t stream) {
  if (!desc || desc->size != sizeof(hipgemm_moe_desc)) return hipErrorInvalidValue;
  const hipgemm_moe_desc& d = *desc;
  const bool e4m3 = d.format == HIPGEMM_W8_E4M3;
  if (d.T < 0 || d.k < 1 || d.k > 64 || d.E < 1 || d.E > HIPGEMM_MOE_MAX_EXPERTS || d.D < 32 ||
      d.F < 32 || d.D % 32 != 0 || d.F % 32 != 0 || d.D > kMaxDim || d.F > kMaxDim / 2 ||
      d.format < 0 || d.format > HIPGEMM_W8_E4M3 ||
      (d.x_type != HIPGEMM_IN_BF16 && d.x_type != HIPGEMM_IN_F16) || d.out_dtype < 0 ||
      d.out_dtype > HIPGEMM_OUT_F32 || d.activation < 0 || d.activation > HIPGEMM_ACT_SILU)
    return hipErrorInvalidValue;
  if (e4m3 ? d.scale_type != HIPGEMM_IN_F32
           : d.scale_type < 0 || d.scale_type > HIPGEMM_SCALE_E8M0 || d.group_size <= 0 ||
                 d.group_size % 32 != 0)
    return hipErrorInvalidValue;
  if (d.T == 0) return hipSuccess;
  if (!d.x || !d.ids || !d.weights || !d.y || !aligned(d.x, 16) || !aligned(d.ids, 4) ||
      !aligned(d.weights, 4) || !aligned(d.y, out_bytes(d.out_dtype)) || d.ldx < d.D ||
      d.ldx % 8 != 0 || d.ldy < d.D || !matrix_ok(d.w13, 2 * d.F, d.D, d) ||
      !matrix_ok(d.w2, d.D, d.F, d))
    return hipErrorInvalidValue;
  if (!d.workspace || !aligned(d.workspace, 16) ||
      d.workspace_bytes < hipgemm_moe_workspace_size(d.T, d.k, d.E, d.D, d.F))
    return hipErrorInvalidValue;

  MoeArgs g{};
  const int ss = type_bytes(d.scale_type), ys = out_bytes(d.out_dtype);
  g.w13 = static_cast<const uint8_t*>(d.w13.weight);
  g.s13 = static_cast<const uint8_t*>(d.w13.scales);
  g.z13 = d.w13.zeros;
  g.w2 = static_cast<const uint8_t*>(d.w2.weight);
  g.s2 = static_cast<const uint8_t*>(d.w2.scales);
  g.z2 = d.w2.zeros;
  g.ldx = 2 * d.ldx;
  g.ldy = d.ldy;
  g.w13_row = d.w13.ldw;
  g.w13_expert = d.w13.expert_w;
  g.s13_row = d.w13.lds * ss;
  g.s13_expert = d.w13.expert_s * ss;
  g.z13_row = d.w13.lds;
  g.z13_expert = d.w13.expert_s;
  g.w2_row = d.w2.ldw;
  g.w2_expert = d.w2.expert_w;
  g.s2_row = d.w2.lds * ss;
  g.s2_expert = d.w2.expert_s * ss;
  g.z2_row = d.w2.lds;
  g.z2_expert = d.w2.expert_s;
  g.k = d.k;
  g.E = d.E;
  g.D = d.D;
  g.F = d.F;
  g.G = e4m3 ? 32 : d.group_size;
  g.act = d.activation;
  g.out = d.out_dtype;
  g.h_parts = h_parts(d.out_dtype);
  const int most = turn_tokens(d.T, d.k);
  g.h = static_cast<uint16_t*>(d.workspace);
  g.o = reinterpret_cast<float*>(g.h + (size_t)most * d.k * 3 * d.F);
  for (int t = 0; t < d.T; t += most) {
    g.T = d.T - t < most ? d.T - t : most;
    g.x = static_cast<const uint8_t*>(d.x) + (long long)t * g.ldx;
    g.ids = d.ids + (long long)t * d.k;
    g.weights = d.weights + (long long)t * d.k;
    g.y = static_cast<uint8_t*>(d.y) + (long long)t * d.ldy * ys;
    const hipError_t e = turn(g, d, stream);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
