// Instantiations of the kernels with 4-bit weights for one activation type and
// weight format (kw4_*.hip).
#pragma once

#include "kernels.hpp"

#include "hipgemm/detail/w4_rows.hpp"

namespace hipgemm {
namespace kernels {

template <class F>
const void* sel_scale(int s, F&& f) {
  return sel4(s, f);
}

template <int kX, int kW>
const void* w4_vec_of(int s, int rows) {
  using namespace detail;
  return sel_scale(s, [&](auto S) -> const void* {
    constexpr int kS = decltype(S)::value;
    switch (rows) {
      case 1: return (const void*)&k_w4_vec<kX, kW, kS, 1>;
      case 2: return (const void*)&k_w4_vec<kX, kW, kS, 2>;
      case 4: return (const void*)&k_w4_vec<kX, kW, kS, 4>;
      default: return nullptr;
    }
  });
}

template <int kX, int kW>
const void* w4_rows_of(int s, int mode, int mt) {
  using namespace detail;
  return sel_scale(s, [&](auto S) -> const void* {
    constexpr int kS = decltype(S)::value;
    // fp4 with E8M0 scales and bf16 activations takes kInline alone.
    constexpr bool kOnlyInline = kX == kInBf16 && kW == kWFp4 && kS == kScaleE8M0;
    auto by_mt = [&](auto Mode) -> const void* {
      constexpr int kMode = decltype(Mode)::value;
      switch (mt) {
        case 1: return (const void*)&k_w4_rows<kX, kW, kS, kMode, 2, 1>;
        case 2: return (const void*)&k_w4_rows<kX, kW, kS, kMode, 2, 2>;
        default: return nullptr;
      }
    };
    if constexpr (kOnlyInline) {
      return mode == kInline ? by_mt(ic<kInline>{}) : nullptr;
    } else {
      return mode == kCoarse ? by_mt(ic<kCoarse>{}) : mode == kFine ? by_mt(ic<kFine>{}) : nullptr;
    }
  });
}

}  // namespace kernels
}  // namespace hipgemm
