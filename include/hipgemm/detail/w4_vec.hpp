// Products of up to four rows of 16-bit activations with 4-bit weights:
// y[m, n] = act(sum_k x[m, k] w[n, k] + bias[n]).
//
// A pass over the weights: each wave takes a chunk of 32 * lk codes of K (lk
// lanes of 16 bytes, so one load reads lk * 16 consecutive bytes of a row; 1 KiB
// at the usual 64), holds the activations of its chunk in registers, and runs
// down kVecSteps rows with them.  So a weight costs its own load and nothing
// else (the matrix unit's tiles would ask for a load of activations per load of
// weights), and a lane's 32 codes lie in one scale group, whose scale multiplies
// the lane's partial sum.  Products by the two-element dot instructions in
// fp32.  Chunks are dealt to the waves_k waves of a row group; partial sums meet
// in a transposed butterfly over the lanes (rows are halved as lanes are: 10
// exchanges for 8 rows instead of 48) and then in LDS.
//
// The int4 excess (decode.hpp) is (bias + z) times the lane's sum of x.  Where
// x is so large that the unscaled sums could overflow, or infinite, the wave
// takes its weights one by one instead, so that infinities come out as the
// definition has them.
#pragma once

#include "decode.hpp"
#include "epilogue.hpp"

namespace hipgemm {
namespace detail {

// Arguments of the kernels with 4-bit weights.  Strides in bytes, but ldy in
// elements.
struct W4Args {
  const uint8_t* x;
  const uint8_t* w;
  const uint8_t* s;
  const uint8_t* z;  // or null (8)
  uint8_t* y;
  const float* bias;  // or null
  long long ldx, ldw, lds, ldz, ldy;
  int M, N, K, G;
  int act, out;
  int lk, waves_k;  // k_w4_vec only
};

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case kActRelu: return relu(v);
    case kActGeluTanh: return gelu_tanh(v);
    case kActSilu: return silu(v);
    default: return v;
  }
}

// One result, rounded to nearest even.
__device__ __forceinline__ void store_result(uint8_t* y, long long i, int out, float v) {
  if (out == kOutF32) reinterpret_cast<float*>(y)[i] = v;
  else if (out == kOutF16) reinterpret_cast<_Float16*>(y)[i] = (_Float16)v;
  else reinterpret_cast<__bf16*>(y)[i] = (__bf16)v;
}

constexpr int kVecSteps = 8;

// One lane's 32 weights (at w) times its 32 activations, one by one and scaled
// first.
template <int kX, int kW>
__device__ __forceinline__ float slow_dot32(const uint8_t* x, const uint8_t* w, float s, float z) {
  float sum = 0.0f;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const uint32_t c = w[i];
    const f32x2 v = unpack2<kX>(reinterpret_cast<const uint32_t*>(x)[i]);
    sum = __builtin_fmaf(v[0], s * code_value<kW>(c & 15u, z), sum);
    sum = __builtin_fmaf(v[1], s * code_value<kW>(c >> 4, z), sum);
  }
  return sum;
}

// Magnitudes of x whose products with codes, and their sums, cannot overflow.
constexpr float kSafeSum = 0x1p112f;

template <int kX, int kW, int kS, int kM>
__global__ __launch_bounds__(512) void k_w4_vec(W4Args g) {
  const int wave = wave_id(), lane = lane_id();
  const int lk = g.lk, per = kWave / lk;  // rows per step
  const int wk = wave % g.waves_k, wr = wave / g.waves_k;
  const int waves_r = (int)(blockDim.x / kWave) / g.waves_k;
  const int rows = kVecSteps * per;  // of a wave
  const int row0 = ((int)blockIdx.x * waves_r + wr) * rows;
  const int kl = lane & (lk - 1), rl = lane / lk;

  float acc[kM][kVecSteps] = {};
  for (int k0 = (wk * lk + kl) * 32; k0 - kl * 32 < g.K; k0 += g.waves_k * lk * 32) {
    const bool in = k0 < g.K;
    // Weights, scales and zero points of this chunk's rows first: all of them
    // are in flight while the activations are read.
    i32x4 w[kVecSteps];
    float s[kVecSteps], z[kVecSteps];
    const unsigned grp = in ? (unsigned)k0 / (unsigned)g.G : 0u;
#pragma unroll
    for (int i = 0; i < kVecSteps; ++i) {
      const int r = min(row0 + i * per + rl, g.N - 1);
      w[i] = in ? __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(
                      g.w + r * g.ldw + (k0 >> 1)))
                : i32x4{};
    }
#pragma unroll
    for (int i = 0; i < kVecSteps; ++i) {
      const int r = min(row0 + i * per + rl, g.N - 1);
      s[i] = scale_at<kS>(g.s + r * g.lds, grp);
      if constexpr (kW == kWInt4) z[i] = g.z ? (float)g.z[r * g.ldz + grp] : 8.0f;
      else z[i] = 0.0f;
    }
    i32x4 x[kM][4];
    float xs[kM];
    bool odd = false;
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      const uint8_t* p = g.x + min(m, g.M - 1) * g.ldx + 2ll * k0;
      xs[m] = 0.0f;
      float mag = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const i32x4 v = in ? reinterpret_cast<const i32x4*>(p)[j] : i32x4{};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (kW == kWInt4) xs[m] = dot2<kX>((uint32_t)v[e], kOnes2<kX>, xs[m]);
          const f32x2 f = unpack2<kX>((uint32_t)v[e]);
          mag = fmaxf(mag, fmaxf(__builtin_fabsf(f[0]), __builtin_fabsf(f[1])));
        }
        x[m][j] = pair_order<kW>(v);
      }
      // (fp16 stays below it unless infinite; the maximum ignores a NaN, which
      // comes out as one either way)
      odd |= !(mag < kSafeSum);
    }
    const bool any_odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    if (!any_odd) {
#pragma unroll
      for (int i = 0; i < kVecSteps; ++i) {
        float d[kM] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const i32x4 b = decode8<kX, kW>((uint32_t)w[i][j], 0u, 1.0f);
#pragma unroll
          for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              d[m] = dot2<kX>((uint32_t)x[m][j][e], (uint32_t)b[e], d[m]);
        }
#pragma unroll
        for (int m = 0; m < kM; ++m) {
          if constexpr (kW == kWInt4)
            d[m] = __builtin_fmaf(-(kInt4Bias<kX> + z[i]), xs[m], d[m]);
          if (in) acc[m][i] = __builtin_fmaf(s[i], d[m], acc[m][i]);
        }
        sched_fence();  // one step's decoded codes at a time in registers
      }
    } else if (in) {
#pragma unroll 1
      for (int i = 0; i < kVecSteps; ++i) {
        const int r = min(row0 + i * per + rl, g.N - 1);
        const float sc = scale_at<kS>(g.s + r * g.lds, grp);
        const float zp = g.z ? (float)g.z[r * g.ldz + grp] : 8.0f;
#pragma unroll
        for (int m = 0; m < kM; ++m) {
          const float v = slow_dot32<kX, kW>(g.x + min(m, g.M - 1) * g.ldx + 2ll * k0,
                                             g.w + r * g.ldw + (k0 >> 1), sc, zp);
#pragma unroll
          for (int e = 0; e < kVecSteps; ++e) acc[m][e] = e == i ? acc[m][e] + v : acc[m][e];
        }
      }
    }
  }

  // Sum over the lk lanes of a row: three steps that halve the rows a lane
  // holds (lane bits 0-2 choose the row step), then plain ones.
  __shared__ float part[8 * kVecSteps * 8 * kM];
#pragma unroll
  for (int m = 0; m < kM; ++m) {
    float v[kVecSteps];
#pragma unroll
    for (int i = 0; i < kVecSteps; ++i) v[i] = acc[m][i];
#pragma unroll
    for (int b = 0, n = kVecSteps; b < 3; ++b) {
      n /= 2;
      const bool up = (lane >> b) & 1;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float give = up ? v[i] : v[i + n];
        const float keep = up ? v[i + n] : v[i];
        v[i] = keep + __shfl_xor(give, 1 << b, kWave);
      }
    }
    for (int b = 8; b < lk; b *= 2) v[0] += __shfl_xor(v[0], b, kWave);
    // Lane bits 0, 1, 2 are bits 2, 1, 0 of the step whose row it holds.
    if (kl < 8) {
      const int step = ((kl & 1) << 2) | (kl & 2) | ((kl >> 2) & 1);
      part[((wr * g.waves_k + wk) * kM + m) * rows + step * per + rl] = v[0];
    }
  }
  __syncthreads();
  const int total = waves_r * kM * rows;
  for (int i = threadIdx.x; i < total; i += blockDim.x) {
    const int r = i % rows, m = i / rows % kM, q = i / (rows * kM);
    const int n = ((int)blockIdx.x * waves_r + q) * rows + r;
    float v = 0.0f;
    for (int w = 0; w < g.waves_k; ++w) v += part[((q * g.waves_k + w) * kM + m) * rows + r];
    if (n < g.N && m < g.M) {
      if (g.bias) v += g.bias[n];
      store_result(g.y, m * g.ldy + n, g.out, activate(v, g.act));
    }
  }
}

}  // namespace detail
}  // namespace hipgemm
