// hipgemm_w4_gemm: arguments, the choice of kernel and its launch.
#include "hipgemm.h"

#include "kernels.hpp"

#include "hipgemm/detail/w4_vec.hpp"
#include "hipgemm/detail/w4_stream.hpp"

namespace hipgemm {
namespace kernels {

const void* w4_vec_bf16_int4(int s, int rows);
const void* w4_vec_bf16_fp4(int s, int rows);
const void* w4_vec_f16_int4(int s, int rows);
const void* w4_vec_f16_fp4(int s, int rows);
const void* w4_rows_bf16_int4(int s, int mode, int mt);
const void* w4_rows_bf16_fp4(int s, int mode, int mt);
const void* w4_rows_f16_int4(int s, int mode, int mt);
const void* w4_rows_f16_fp4(int s, int mode, int mt);

const void* w4_vec(int x, int w, int s, int rows) {
  if (x == detail::kInBf16)
    return w == detail::kWInt4 ? w4_vec_bf16_int4(s, rows) : w4_vec_bf16_fp4(s, rows);
  return w == detail::kWInt4 ? w4_vec_f16_int4(s, rows) : w4_vec_f16_fp4(s, rows);
}
const void* w4_rows(int x, int w, int s, int mode, int mt) {
  if (x == detail::kInBf16)
    return w == detail::kWInt4 ? w4_rows_bf16_int4(s, mode, mt) : w4_rows_bf16_fp4(s, mode, mt);
  return w == detail::kWInt4 ? w4_rows_f16_int4(s, mode, mt) : w4_rows_f16_fp4(s, mode, mt);
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

hipError_t launch(const void* fn, dim3 grid, int threads, W4Args& g, hipStream_t stream) {
  if (!fn) return hipErrorInvalidValue;
  void* args[] = {&g};
  return hipLaunchKernel(fn, grid, dim3((unsigned)threads), args, 0, stream);
}

// Lanes along K of a step, waves along K and rows of a workgroup.  lk: the
// widest that leaves few lanes without codes in the last chunk.
void vec_shape(int K, int* lk, int* waves_k, int* waves_r) {
  const int units = K / 32;
  int best = 64;
  for (int l = 64; l >= 8; l /= 2) {
    const int covered = (units + l - 1) / l * l, least = (units + best - 1) / best * best;
    if (covered * 5 < least * 4) best = l;
  }
  const int chunks = units > best ? (units + best - 1) / best : 1;
  const int turns = (chunks + 7) / 8;
  *lk = best;
  *waves_k = (chunks + turns - 1) / turns;
  *waves_r = *waves_k >= 4 ? 1 : 4 / *waves_k;
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
  if (d.M <= 4) {
    int waves_r;
    vec_shape(d.K, &g.lk, &g.waves_k, &waves_r);
    const int rows = kVecSteps * (kWave / g.lk) * waves_r;
    return launch(hk::w4_vec(d.x_type, d.format, d.scale_type, d.M == 3 ? 4 : d.M),
                  dim3((unsigned)((d.N + rows - 1) / rows)), kWave * g.waves_k * waves_r, g,
                  stream);
  }
  const int mode = d.format == HIPGEMM_W4_FP4 && d.scale_type == HIPGEMM_SCALE_E8M0 &&
                           d.x_type == HIPGEMM_IN_BF16
                       ? kInline
                   : d.group_size % 128 == 0 ? kCoarse
                                             : kFine;
  const int mt = d.M <= 16 ? 1 : 2;
  const unsigned tiles_m = (unsigned)((d.M + 16 * mt - 1) / (16 * mt));
  return launch(hk::w4_rows(d.x_type, d.format, d.scale_type, mode, mt),
                dim3((unsigned)((d.N + 31) / 32), tiles_m), 512, g, stream);
}

}  // namespace

extern "C" hipError_t hipgemm_w4_gemm(const hipgemm_w4_desc* desc, hipStream_t stream) {
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
        d.lds < (d.K + d.group_size - 1) / d.group_size)
      return hipErrorInvalidValue;
  }
  return run(d, stream);
}
