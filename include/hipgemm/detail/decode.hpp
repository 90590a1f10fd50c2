// Quantised weights as 16-bit MFMA operands, for products with 16-bit
// activations: int4 and fp4 (E2M1) with one scale per group along K, and e4m3.
//
// Decoding is exact: every code's value has at most 8 significand bits, so it
// is a bf16 and an fp16 number, and scales are applied in fp32 after the
// products.  int4 codes (0-15, value q - z) come out as q: a nibble is the e4m3
// number q 2^-9 (subnormal below 8, the first binade from there), so unpacked
// nibbles go through the e4m3 conversion with scale 2^9, nine instructions for
// eight.  The excess is z times the sum of x over the group, formed once per group
// and row of x and subtracted in fp32.  (Seven instructions give q + 128 in bf16, out
// of order, with an excess sixteen times as large: errors of 5e-7 of the results'
// rms at K = 4096 for 8e-8, one row of 28672 x 8192 24.5 us for 24.2, and 64 tokens
// of 8 of 128 experts of 4096 x 1536 263 for 267.)
#pragma once

#include "arch.hpp"

namespace hipgemm {
namespace detail {

using bf16x8_t = __bf16 __attribute__((ext_vector_type(8)));
using f16x8_t = _Float16 __attribute__((ext_vector_type(8)));
using f16x2_t = _Float16 __attribute__((ext_vector_type(2)));

// Types of activations and scales (HIPGEMM_IN_* and HIPGEMM_SCALE_E8M0).
constexpr int kInF32 = 0, kInBf16 = 1, kInF16 = 2, kScaleE8M0 = 3;
__host__ __device__ constexpr int type_bytes(int t) {
  return t == kInF32 ? 4 : t == kScaleE8M0 ? 1 : 2;
}
// Weight formats (HIPGEMM_W4_*, HIPGEMM_W8_E4M3; int4 with zero points is a
// format of its own to the kernels).
constexpr int kWInt4 = 0, kWFp4 = 1, kWE4M3 = 2, kWInt4Z = 3;
__host__ __device__ constexpr bool is_int4(int w) { return w == kWInt4 || w == kWInt4Z; }

template <int kX>
__device__ __forceinline__ f32x4 mfma_16x16x32(i32x4 a, i32x4 b, f32x4 c) {
  if constexpr (kX == kInBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(
        __builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// a.lo * b.lo + a.hi * b.hi + c of two packed pairs, in fp32.
template <int kX>
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
  if constexpr (kX == kInBf16)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, a),
                                           __builtin_bit_cast(bf16x2_t, b), c, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, a),
                                  __builtin_bit_cast(f16x2_t, b), c, false);
}

// One packed pair as two floats.
template <int kX>
__device__ __forceinline__ f32x2 unpack2(uint32_t a) {
  if constexpr (kX == kInBf16)
    return f32x2{__builtin_bit_cast(float, a << 16),
                 __builtin_bit_cast(float, a & 0xffff0000u)};
  const f16x2_t h = __builtin_bit_cast(f16x2_t, a);
  return f32x2{(float)h[0], (float)h[1]};
}

// 1.0 twice.
template <int kX>
constexpr uint32_t kOnes2 = kX == kInBf16 ? 0x3f803f80u : 0x3c003c00u;

// A scale as fp32, from its bits.  E8M0: 2^(e - 127), 255 is NaN.
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
template <int kS>
__device__ __forceinline__ float scale_at(const void* p, long long i) {
  if constexpr (type_bytes(kS) == 4) return scale_of<kS>(static_cast<const uint32_t*>(p)[i]);
  else if constexpr (type_bytes(kS) == 2) return scale_of<kS>(static_cast<const uint16_t*>(p)[i]);
  else return scale_of<kS>(static_cast<const uint8_t*>(p)[i]);
}

// Eight codes of a dword (eight bytes for e4m3: lo, hi) as a 16-bit fragment;
// for fp4 and e4m3 times `scale`, a power of two that the result holds exactly.
template <int kX, int kW>
__device__ __forceinline__ i32x4 decode8(uint32_t lo, uint32_t hi, float scale) {
  i32x4 r;
  if constexpr (is_int4(kW)) {
    const uint32_t low = lo & 0x0f0f0f0fu, high = (lo >> 4) & 0x0f0f0f0fu;
    r = decode8<kX, kWE4M3>(__builtin_amdgcn_perm(high, low, 0x05010400u),
                            __builtin_amdgcn_perm(high, low, 0x07030602u), 512.0f);
  } else if constexpr (kW == kWFp4) {
    if constexpr (kX == kInBf16) {
      r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(lo, scale, 0));
      r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(lo, scale, 1));
      r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(lo, scale, 2));
      r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(lo, scale, 3));
    } else {
      r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(lo, scale, 0));
      r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(lo, scale, 1));
      r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(lo, scale, 2));
      r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(lo, scale, 3));
    }
  } else {
    if constexpr (kX == kInBf16) {
      r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
      r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
      r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
      r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    } else {
      r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false));
      r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true));
      r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false));
      r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true));
    }
  }
  return r;
}

// The value of one 4-bit code, scale excluded (rare paths).
template <int kW>
__device__ __forceinline__ float code_value(uint32_t q, float z) {
  if constexpr (is_int4(kW)) return (float)q - z;
  const uint32_t m = q & 7u;
  const float v = m < 2u ? 0.5f * (float)m
                         : __builtin_bit_cast(float, ((126u + (m >> 1)) << 23) | ((m & 1u) << 22));
  return q & 8u ? -v : v;
}

}  // namespace detail
}  // namespace hipgemm
