// The router's choice: for each token the k experts of largest logit, and their
// weights.
//
// Ordering: logits become 32-bit keys whose unsigned order is theirs (-0 as +0,
// NaN above infinity, -inf as 0: never chosen), kV of them in each of a token's
// kL lanes, neighbours in one lane.  A round takes the lanes' maxima (three at a
// time: v_max3_u32), reduces them over the kL lanes by DPP and clears the key that
// it found; lane j keeps the j-th result.  Equal logits go to the lowest expert:
// keys of 16-bit logits hold it (and so say themselves whose they are), for fp32 it
// is the first lane that has the maximum and its first value.  Weights are then
// computed once, in lanes 0 to k - 1.
//
// What bounds it: one token is the latency of k rounds; many are instructions,
// about 5 kV + 12 per round (16 bits: 3 kV + 12) for 64 / kL tokens at once, so
// that a token's values go to 16 lanes where there are tokens enough to fill the CUs
// (fewer exchanges per value), to all 64 where there are not.  us in a graph: one
// token, 8 of 64, fp32 2.7; 16384 tokens, 8 of 256, bf16 7.2 (9.1 with fp32's keys).
#include "hipgemm.h"

#include "kernels.hpp"

#include "hipgemm/detail/decode.hpp"

namespace hipgemm {
namespace kernels {
namespace {

using namespace detail;

struct RouteArgs {
  const uint8_t* logits;
  float* weights;
  int* ids;
  long long ld;  // bytes
  int T, E, k;
  int sigmoid, renormalize, vec;
  float scale;
};

// fp32: the key is the logit's alone.
__device__ __forceinline__ uint32_t key_of(float f) {
  f += 0.0f;  // -0 -> +0
  uint32_t b = __builtin_bit_cast(uint32_t, f);
  if (f != f) b = 0x7fc00000u;
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return f == -__builtin_inff() ? 0u : b;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  const uint32_t b = key & 0x80000000u ? key & 0x7fffffffu : ~key;
  return key == 0u ? -__builtin_inff() : __builtin_bit_cast(float, b);
}

// 16 bits: the logit's order above, 0xffff - expert below, so that no two keys of a
// token are equal but 0.
template <int kType>
__device__ __forceinline__ uint32_t key16_of(uint32_t b, int e) {
  constexpr uint32_t kInf = kType == kInBf16 ? 0x7f80u : 0x7c00u;
  const uint32_t mag = b & 0x7fffu;
  const bool never = b == (0x8000u | kInf);
  b = mag == 0u ? 0u : mag > kInf ? 0x7fffu : b;
  b ^= b & 0x8000u ? 0xffffu : 0x8000u;
  return never ? 0u : b << 16 | (0xffffu - (uint32_t)e);
}
template <int kType>
__device__ __forceinline__ float value_of(uint32_t key) {
  if constexpr (kType == kInF32) {
    return value_of(key);
  } else {
    const uint32_t o = key >> 16, b = o & 0x8000u ? o & 0x7fffu : o ^ 0xffffu;
    const float f = kType == kInBf16 ? __builtin_bit_cast(float, b << 16)
                                     : (float)__builtin_bit_cast(_Float16, (uint16_t)b);
    return key == 0u ? -__builtin_inff() : f;
  }
}

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xf, 0xf, true);
}
// All lanes of a group of kL (16 or 64) get op over the group: exchanges with
// the neighbour, the pair, the mirrored half row and the mirrored row, then with
// the other rows.
template <int kL, class F>
__device__ __forceinline__ uint32_t all_lanes(uint32_t v, F&& op) {
  v = op(v, dpp<0xb1>(v));   // quad_perm 1, 0, 3, 2
  v = op(v, dpp<0x4e>(v));   // quad_perm 2, 3, 0, 1
  v = op(v, dpp<0x141>(v));  // row_half_mirror
  v = op(v, dpp<0x140>(v));  // row_mirror
  if constexpr (kL == 64) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(b[0], b[1]);
  }
  return v;
}
template <int kL>
__device__ __forceinline__ float sum_lanes(float f) {
  return __builtin_bit_cast(
      float, all_lanes<kL>(__builtin_bit_cast(uint32_t, f), [](uint32_t a, uint32_t b) {
        return __builtin_bit_cast(
            uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
      }));
}

template <int kType>
__device__ __forceinline__ uint32_t key_at(const uint8_t* p, int i) {
  if constexpr (kType == kInF32) return key_of(reinterpret_cast<const float*>(p)[i]);
  else return key16_of<kType>(reinterpret_cast<const uint16_t*>(p)[i], i);
}

template <int kType, int kL, int kV>
__global__ __launch_bounds__(256) void k_route(RouteArgs g) {
  constexpr int kBytes = type_bytes(kType), kPer = 16 / kBytes;
  const int gl = (int)threadIdx.x % kL;  // lane of the token's group
  const int t = (int)blockIdx.x * (256 / kL) + (int)threadIdx.x / kL;
  const bool live = t < g.T;
  const uint8_t* p = g.logits + (long long)(live ? t : g.T - 1) * g.ld;
  const int e0 = gl * kV;

  uint32_t key[kV];
  if (kV * kBytes >= 16 && g.vec) {
#pragma unroll
    for (int c = 0; c < kV / kPer; ++c) {
      i32x4 v = {};
      const bool in = e0 + c * kPer < g.E;
      if (in) v = *reinterpret_cast<const i32x4*>(p + (e0 + c * kPer) * kBytes);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        // (an element goes through an integer: bit_cast of a vector element takes element 0)
        uint32_t q;
        if constexpr (kType == kInF32) q = key_of(__builtin_bit_cast(float, (uint32_t)v[i]));
        else q = key16_of<kType>((uint32_t)v[i / 2] >> (16 * (i & 1)) & 0xffffu, e0 + c * kPer + i);
        key[c * kPer + i] = in ? q : 0u;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) key[i] = e0 + i < g.E ? key_at<kType>(p, e0 + i) : 0u;
  }

  auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  uint32_t top = 0;        // the largest key
  float total = 1.0f;      // sum of all exponentials, where it is asked for
  uint32_t mine_key = 0;
  int mine_id = -1;
  for (int j = 0; j < g.k; ++j) {
    uint32_t m = key[0];
#pragma unroll
    for (int i = 1; i < kV; ++i) m = larger(m, key[i]);
    const uint32_t best = all_lanes<kL>(m, larger);
    if (j == 0) {
      top = best;
      if (!g.sigmoid && !g.renormalize) {
        const float ref = value_of<kType>(top);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kV; ++i) s += key[i] ? expf(value_of<kType>(key[i]) - ref) : 0.0f;
        total = sum_lanes<kL>(s);
      }
    }
    int id;
    if constexpr (kType == kInF32) {
      // The first lane of the group whose maximum it is, and its first value.
      const uint64_t has = __builtin_amdgcn_ballot_w64(m == best);
      const int base = lane_id() & ~(kL - 1);
      const uint64_t in_group = kL == 64 ? has : (has >> base) & ((1ull << kL) - 1ull);
      const int owner = __builtin_ctzll(in_group);
      int at = 0;
  #pragma unroll
      for (int i = kV - 1; i >= 0; --i) at = key[i] == best ? i : at;
      const bool own = gl == owner;
  #pragma unroll
      for (int i = 0; i < kV; ++i) key[i] = own && at == i ? 0u : key[i];
      id = owner * kV + __shfl(at, base + owner, kWave);
    } else {
      id = 0xffff - (int)(best & 0xffffu);
#pragma unroll
      for (int i = 0; i < kV; ++i) key[i] = key[i] == best ? 0u : key[i];
    }
    if (gl == j && best != 0u) {
      mine_key = best;
      mine_id = id;
    }
  }

  // Sigmoids that are divided by their sum, of a token whose logits are all negative:
  // each times exp(-max), which the division takes out again.  By themselves they
  // would all be 0 below -88, and 0 / 0 no weight.
  const float v = value_of<kType>(mine_key), ref = value_of<kType>(top);
  const bool sigmoid = g.sigmoid && !(g.renormalize && ref < 0.0f);
  float w = 0.0f;
  if (mine_id >= 0) {
    w = expf(sigmoid ? -v : v - ref);
    if (sigmoid) w = 1.0f / (1.0f + w);
    else if (g.sigmoid) w /= 1.0f + expf(v);
  }
  if (g.renormalize) total = sum_lanes<kL>(w);
  w = mine_id >= 0 ? w / total * g.scale : 0.0f;
  if (live && gl < g.k) {
    g.weights[(long long)t * g.k + gl] = w;
    g.ids[(long long)t * g.k + gl] = mine_id;
  }
}

template <int kType, int kL>
const void* route_of(int v) {
  switch (v) {
    case 1: return (const void*)&k_route<kType, kL, 1>;
    case 2: return (const void*)&k_route<kType, kL, 2>;
    case 4: return (const void*)&k_route<kType, kL, 4>;
    case 8: return (const void*)&k_route<kType, kL, 8>;
    case 16: return (const void*)&k_route<kType, kL, 16>;
    default:
      if constexpr (kL == 16) return v == 32 ? (const void*)&k_route<kType, kL, 32> : nullptr;
      return nullptr;
  }
}
template <int kL>
const void* route_fn(int type, int v) {
  return type == kInF32 ? route_of<kInF32, kL>(v)
                        : type == kInBf16 ? route_of<kInBf16, kL>(v) : route_of<kInF16, kL>(v);
}

}  // namespace
}  // namespace kernels
}  // namespace hipgemm

extern "C" hipError_t hipgemm_moe_route(const void* logits, int type, int T, int E, int k,
                                        long long ld, int scoring, int renormalize, float scale,
                                        float* weights, int* ids, hipStream_t stream) {
  using namespace hipgemm::kernels;
  if (T < 0 || E < 1 || E > HIPGEMM_MOE_MAX_EXPERTS || k < 1 || k > E || k > 64 ||
      type < HIPGEMM_IN_F32 || type > HIPGEMM_IN_F16 ||
      (scoring != HIPGEMM_MOE_SOFTMAX && scoring != HIPGEMM_MOE_SIGMOID))
    return hipErrorInvalidValue;
  if (T == 0) return hipSuccess;
  const int es = type == HIPGEMM_IN_F32 ? 4 : 2;
  auto aligned = [](const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; };
  if (!logits || !weights || !ids || ld < E || !aligned(logits, es) || !aligned(weights, 4) ||
      !aligned(ids, 4))
    return hipErrorInvalidValue;
  RouteArgs g{static_cast<const uint8_t*>(logits), weights, ids, ld * es, T, E, k,
              scoring == HIPGEMM_MOE_SIGMOID, renormalize != 0, 0, scale};
  g.vec = aligned(logits, 16) && g.ld % 16 == 0 && E % (16 / es) == 0;
  // 16 lanes per token from the tokens on that give every SIMD a wave so (4 x
  // 256 SIMDs).
  const bool narrow = k <= 16 && E <= 512 && T >= 4096;
  const int lanes = narrow ? 16 : 64;
  int v = 1;
  while (v * lanes < E) v *= 2;
  const void* fn = narrow ? route_fn<16>(type, v) : route_fn<64>(type, v);
  if (!fn) return hipErrorInvalidValue;
  void* args[] = {&g};
  const int per = 256 / lanes;
  return hipLaunchKernel(fn, dim3((unsigned)((T + per - 1) / per)), dim3(256), args, 0, stream);
}
