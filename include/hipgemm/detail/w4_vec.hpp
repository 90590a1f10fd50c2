// Products of a few rows of 16-bit activations with quantised weights, a pass
// over the weights' rows: y[m, n] = act(sum_k x[m, k] w[n, k] + bias[n]).
//
// Each wave takes a chunk of K, 16 bytes of weights per lane (kLk lanes of a row:
// 1 KiB of one row at the usual 64), holds the activations of its chunk in
// registers, and runs down its rows with them, eight loads at a time and eight
// ahead.  So a weight costs its own load and nothing else (the matrix unit's
// tiles would ask for a read of activations per load of weights), memory is read
// in the longest pieces there are, and a lane's weights lie in one scale group,
// whose scale multiplies the lane's partial sum.  Products by the two-element dot
// instructions in fp32.  The lanes' sums meet in a butterfly that halves the rows
// as it halves the lanes, those of the chunks in LDS.
//
// The int4 excess (decode.hpp) is z times the lane's sum of x.  Where
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
  int waves_k, rows, wave_rows;  // k_w4_vec: of a workgroup, of a wave
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

// Magnitudes of x whose products with codes, and their sums, cannot overflow.
constexpr float kSafeSum = 0x1p112f;
constexpr int kVecRows = 8;       // loads of a step
constexpr int kVecMaxRows = 128;  // of a workgroup

// One wave's part: kM rows of x by rows of one matrix, over one chunk of K.
template <int kX, int kW, int kS, int kM, int kLk>
struct Vec {
  static constexpr int kPer = kWave / kLk;              // rows of a load
  static constexpr int kStep = kVecRows * kPer;         // rows of a step
  static constexpr int kElems = kW == kWE4M3 ? 16 : 32;  // of a lane
  static constexpr int kWords = kElems / 8;
  static constexpr int kChunk = kLk * kElems;
  // (e4m3 rows have one scale each: group 0)
  static constexpr bool kGroups = kW != kWE4M3;

  i32x4 x[kM][kWords];
  float xs[kM];
  bool odd;        // the wave's x is out of the ordinary
  int k;           // this lane's first element, or its last valid start
  bool in;
  uint32_t grp;

  struct Rows {
    i32x4 w[kVecRows];
    uint32_t s[kVecRows], z[kVecRows];
  };

  // The chunk's activations, loaded to v, into the form that dot takes.
  __device__ __forceinline__ void take(i32x4 (&v)[kM][kWords]) {
    bool any = false;
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      float top = 0.0f;
      xs[m] = 0.0f;
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        if (!in) v[m][j] = i32x4{};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t u = (uint32_t)v[m][j][e];
          if constexpr (is_int4(kW)) xs[m] = dot2<kX>(u, kOnes2<kX>, xs[m]);
          if constexpr (kGroups) {
            const f32x2 f = unpack2<kX>(u);
            top = fmaxf(top, fmaxf(__builtin_fabsf(f[0]), __builtin_fabsf(f[1])));
          }
        }
        x[m][j] = v[m][j];
      }
      // (fp16 stays below it unless infinite; the maximum ignores a NaN, which
      // comes out as one either way)
      any |= !(top < kSafeSum);
    }
    odd = kGroups && __builtin_amdgcn_ballot_w64(any) != 0;
  }

  // v, of which the compiler holds nothing that it computed from it before.
  __device__ __forceinline__ static uint32_t anew(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
  }

  // Rows row to below end of a matrix, zeros past end.  Rows are stepped by the lane's
  // offset, which the range check sees, not by the scalar one, which it may leave
  // out: nothing past the matrix' last row is asked of memory.  The sums are made
  // anew at every step (held over the loop they cost 14 registers and with them a
  // wave per SIMD: 15 pairs of fp4 2336 x 1056 took 25.7 us for 23.5).
  __device__ __forceinline__ void load(Rows& r, const uint8_t* w, long long ldw, const uint8_t* s,
                                       long long lds, const uint8_t* z, long long ldz, int row,
                                       int end) const {
    const int left = max(min(end - row, kStep), 0), rl = lane_id() / kLk;
    const auto wb = make_rsrc(w + row * ldw, (uint32_t)(left * ldw));
    const uint32_t wo = anew(in ? (uint32_t)(rl * ldw) + (kW == kWE4M3 ? k : k >> 1) : kOobOffset);
#pragma unroll
    for (int i = 0; i < kVecRows; ++i)
      r.w[i] = __builtin_amdgcn_raw_buffer_load_b128(wb, wo + (uint32_t)(i * kPer * ldw), 0, kStoreC);
    {
      const auto sb = make_rsrc(s + row * lds, (uint32_t)(left * lds));
      const uint32_t so = anew((uint32_t)(rl * lds) + grp * type_bytes(kS));
#pragma unroll
      for (int i = 0; i < kVecRows; ++i) {
        const uint32_t at = so + (uint32_t)(i * kPer * lds);
        if constexpr (type_bytes(kS) == 4) r.s[i] = __builtin_amdgcn_raw_buffer_load_b32(sb, at, 0, 0);
        else if constexpr (type_bytes(kS) == 2)
          r.s[i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(sb, at, 0, 0);
        else r.s[i] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(sb, at, 0, 0);
      }
      if constexpr (kW == kWInt4Z) {
        const auto zb = make_rsrc(z + row * ldz, (uint32_t)(left * ldz));
        const uint32_t zo = anew((uint32_t)(rl * ldz) + grp);
#pragma unroll
        for (int i = 0; i < kVecRows; ++i)
          r.z[i] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(zb, zo + (uint32_t)(i * kPer * ldz), 0, 0);
      }
    }
  }

  // The lane's sums over its part of the chunk.
  template <class F>
  __device__ __forceinline__ void dot(const Rows& r, int K, F&& xr, float (&sum)[kM][kVecRows]) const {
#pragma unroll
    for (int i = 0; i < kVecRows; ++i) {
      float d[kM] = {};
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        const i32x4 b = kW == kWE4M3
                            ? decode8<kX, kW>((uint32_t)r.w[i][2 * j % 4], (uint32_t)r.w[i][(2 * j + 1) % 4], 1.0f)
                            : decode8<kX, kW>((uint32_t)r.w[i][j], 0u, 1.0f);
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            d[m] = dot2<kX>((uint32_t)x[m][j][e], (uint32_t)b[e], d[m]);
      }
      const float sc = scale_of<kS>(r.s[i]);
      float off = -8.0f;
      if constexpr (kW == kWInt4Z) off = -(float)r.z[i];
#pragma unroll
      for (int m = 0; m < kM; ++m) {
        if constexpr (is_int4(kW)) d[m] = __builtin_fmaf(off, xs[m], d[m]);
        sum[m][i] = in ? sc * d[m] : 0.0f;
      }
      sched_fence();  // one row's decoded weights at a time in registers
    }
    // (Not as an else: that would make the loop's branches ones on the lanes.)
    if (__builtin_amdgcn_readfirstlane((int)odd)) {
      // One by one, and scaled first.
#pragma unroll
      for (int i = 0; i < kVecRows; ++i) {
        const float sc = scale_of<kS>(r.s[i]);
        const float z = kW == kWInt4Z ? (float)r.z[i] : 8.0f;
#pragma unroll
        for (int m = 0; m < kM; ++m) {
          float d = 0.0f;
          if (in) {
#pragma unroll 1
            for (int j = 0; j < kElems / 2; ++j) {
              const uint32_t q = (uint32_t)(j < 4 ? r.w[i][0] : j < 8 ? r.w[i][1] : j < 12 ? r.w[i][2] : r.w[i][3]);
              const uint32_t c = q >> (8 * (j & 3)) & 255u;
              const f32x2 v = unpack2<kX>(*reinterpret_cast<const uint32_t*>(xr(m) + 2ll * k + 4 * j));
              d = __builtin_fmaf(v[0], sc * code_value<kW>(c & 15u, z), d);
              d = __builtin_fmaf(v[1], sc * code_value<kW>(c >> 4, z), d);
            }
          }
          sum[m][i] = d;
        }
      }
    }
  }

  // Adds the rows' sums over the lanes to to[row of the step].
  __device__ __forceinline__ void gather(float (&v)[kVecRows], float* to) const {
    const int lane = lane_id();
    if constexpr (kLk == 64) {
      // Half of the rows to the other 32 lanes, half of those to the other 16.
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v[i]),
                                                        __builtin_bit_cast(uint32_t, v[i + 4]), false, false);
        v[i] = __builtin_bit_cast(float, (uint32_t)p[0]) + __builtin_bit_cast(float, (uint32_t)p[1]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v[i]),
                                                        __builtin_bit_cast(uint32_t, v[i + 2]), false, false);
        v[i] = __builtin_bit_cast(float, (uint32_t)p[0]) + __builtin_bit_cast(float, (uint32_t)p[1]);
      }
    }
    constexpr int kLeft = kLk == 64 ? 2 : kVecRows;
#pragma unroll
    for (int i = 0; i < kLeft; ++i) {
      v[i] += dpp_f<0xb1>(v[i]);   // quad_perm 1, 0, 3, 2
      v[i] += dpp_f<0x4e>(v[i]);   // quad_perm 2, 3, 0, 1
      v[i] += dpp_f<0x141>(v[i]);  // row_half_mirror
      v[i] += dpp_f<0x140>(v[i]);  // row_mirror
    }
    if ((lane & 15) == 0) {
#pragma unroll
      for (int i = 0; i < kLeft; ++i) {
        // 64 lanes: lane bit 5 is bit 2 of the row, bit 4 bit 1.  16: rows i kPer + l / 16.
        const int row = kLk == 64 ? i + 2 * (lane >> 4 & 1) + 4 * (lane >> 5) : i * kPer + (lane >> 4);
        to[row] += v[i];
      }
    }
  }
  template <int kCtrl>
  __device__ __forceinline__ static float dpp_f(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                         0, __builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, true));
  }

  // Rows r0 to below r1 of one matrix (rows of K) by the chunk at k0 of the rows
  // of x, xr(m); adds to to[m * kVecMaxRows + row - r0], which is this wave's own.
  template <class F>
  __device__ __forceinline__ void pass(int k0, int K, int group, F&& xr, const uint8_t* w,
                                       long long ldw, const uint8_t* s, long long lds,
                                       const uint8_t* z, long long ldz, int r0, int r1, float* to) {
    k = k0 + (lane_id() & (kLk - 1)) * kElems;
    in = k < K;
    grp = kGroups ? (uint32_t)group_of(min(k, K - 32) >> 5, 32.0f / (float)group) : 0u;
    i32x4 v[kM][kWords];
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int j = 0; j < kWords; ++j)
        v[m][j] = *reinterpret_cast<const i32x4*>(xr(m) + 2ll * min(k + 8 * j, K - 8));
    sched_fence();
    Rows ring[2];
    load(ring[0], w, ldw, s, lds, z, ldz, r0, r1);
    sched_fence();
    take(v);
    for (int row = r0; row < r1; row += 2 * kStep) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = row + u * kStep;
        if (at >= r1) break;
        load(ring[1 - u], w, ldw, s, lds, z, ldz, at + kStep, r1);
        float sum[kM][kVecRows];
        dot(ring[u], K, xr, sum);
#pragma unroll
        for (int m = 0; m < kM; ++m) gather(sum[m], to + m * kVecMaxRows + at - r0);
      }
    }
  }
};

template <int kX, int kW, int kS, int kM, int kLk>
__global__ __launch_bounds__(512) void k_w4_vec(W4Args g) {
  using V = Vec<kX, kW, kS, kM, kLk>;
  const int wave = wave_id(), tid = (int)threadIdx.x;
  const int wk = wave % g.waves_k, wr = wave / g.waves_k;
  // A workgroup's rows, and this wave's.
  const int n0 = (int)blockIdx.x * g.rows;
  const int r0 = n0 + wr * g.wave_rows, r1 = min(min(r0 + g.wave_rows, n0 + g.rows), g.N);
  __shared__ float part[8][kM * kVecMaxRows];
  for (int i = tid; i < 8 * kM * kVecMaxRows; i += (int)blockDim.x) (&part[0][0])[i] = 0.0f;
  __syncthreads();
  auto xr = [&](int m) { return g.x + min(m, g.M - 1) * g.ldx; };
  V v;
  for (int k0 = wk * V::kChunk; k0 < g.K; k0 += g.waves_k * V::kChunk) {
    if (r0 < r1)
      v.pass(k0, g.K, g.G, xr, g.w, g.ldw, g.s, g.lds, g.z, g.ldz, r0, r1, part[wave]);
  }
  __syncthreads();
  for (int i = tid; i < kM * g.rows; i += (int)blockDim.x) {
    const int r = i % g.rows, m = i / g.rows, n = n0 + r;
    if (n >= g.N || m >= g.M) continue;
    const int q = r / g.wave_rows;
    float f = 0.0f;
    for (int w = 0; w < g.waves_k; ++w)
      f += part[q * g.waves_k + w][m * kVecMaxRows + r - q * g.wave_rows];
    if (g.bias) f += g.bias[n];
    store_result(g.y, m * g.ldy + n, g.out, activate(f, g.act));
  }
}

}  // namespace detail
}  // namespace hipgemm
