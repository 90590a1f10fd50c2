// Instantiations of the experts' kernels for one weight format (kmoe_*.hip).
#pragma once

#include "kernels.hpp"

#include "hipgemm/detail/moe.hpp"

namespace hipgemm {
namespace kernels {

// Calls f(scale type, mode) with the combination's constants where it is built:
// e4m3 has row scales, fp4 with E8M0 scales and bf16 activations kInline alone.
template <int kX, int kW, class F>
const void* moe_sel(int s, int mode, F&& f) {
  using namespace detail;
  if constexpr (kW == kWE4M3) {
    return s == kInF32 && mode == kNone ? f(ic<kInF32>{}, ic<kNone>{}) : nullptr;
  } else {
    return sel4(s, [&](auto S) -> const void* {
      if constexpr (kX == kInBf16 && kW == kWFp4 && decltype(S)::value == kScaleE8M0)
        return mode == kInline ? f(S, ic<kInline>{}) : nullptr;
      else
        return mode == kCoarse ? f(S, ic<kCoarse>{}) : mode == kFine ? f(S, ic<kFine>{}) : nullptr;
    });
  }
}

template <int kX, int kW>
const void* moe_up_of(int s, int mode, int mt) {
  return moe_sel<kX, kW>(s, mode, [&](auto S, auto Mode) -> const void* {
    constexpr int kS = decltype(S)::value, kMode = decltype(Mode)::value;
    return mt == 1 ? (const void*)&detail::k_moe_up<kX, kW, kS, kMode, 1>
                   : (const void*)&detail::k_moe_up<kX, kW, kS, kMode, 2>;
  });
}

template <int kW>
const void* moe_down_of(int s, int mode) {
  return moe_sel<detail::kInBf16, kW>(s, mode, [&](auto S, auto Mode) -> const void* {
    return (const void*)&detail::k_moe_down<kW, decltype(S)::value, decltype(Mode)::value>;
  });
}

}  // namespace kernels
}  // namespace hipgemm
