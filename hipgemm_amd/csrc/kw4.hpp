// Instantiations of the kernels with quantised weights and 16-bit activations
// for one weight format (kw4_*.hip, kmoe_*.hip).
#pragma once

#include "kernels.hpp"

#include "hipgemm/detail/moe_vec.hpp"
#include "hipgemm/detail/w4_tile.hpp"

namespace hipgemm {
namespace kernels {

// f(scale type, mode) with the combination's constants, where it is built: e4m3
// has row scales; fp4 with E8M0 scales and bf16 activations takes kInline alone.
template <int kX, int kW, class F>
const void* sel_scales(int s, int mode, F&& f) {
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
const void* w4_vec_of(int s, int rows, int lk) {
  using namespace detail;
  return sel4(s, [&](auto S) -> const void* {
    constexpr int kS = decltype(S)::value;
    auto by_lk = [&](auto M) {
      constexpr int kM = decltype(M)::value;
      return lk == 64 ? (const void*)&k_w4_vec<kX, kW, kS, kM, 64>
                      : (const void*)&k_w4_vec<kX, kW, kS, kM, 16>;
    };
    return rows == 1 ? by_lk(ic<1>{}) : rows == 2 ? by_lk(ic<2>{}) : by_lk(ic<4>{});
  });
}

// f(tiles of 16 rows of x).
template <class F>
const void* sel_mt(int mt, F&& f) {
  return mt == 1 ? f(ic<1>{}) : mt == 2 ? f(ic<2>{}) : nullptr;
}

template <int kX, int kW>
const void* w4_tile_of(int s, int mode) {
  return sel_scales<kX, kW>(s, mode, [](auto S, auto Mode) {
    return (const void*)&detail::k_w4_tile<kX, kW, decltype(S)::value, decltype(Mode)::value>;
  });
}

template <int kX, int kW>
const void* w4_split_of(int s, int mode, int mt, int nt) {
  return sel_scales<kX, kW>(s, mode, [mt, nt](auto S, auto Mode) -> const void* {
    constexpr int kS = decltype(S)::value, kMode = decltype(Mode)::value;
    switch (mt) {
      case 1: return nt == 2 ? (const void*)&detail::k_w4_split<kX, kW, kS, kMode, 1, 2>
                            : (const void*)&detail::k_w4_split<kX, kW, kS, kMode, 1, 4>;
      case 2: return nt == 2 ? (const void*)&detail::k_w4_split<kX, kW, kS, kMode, 2, 2>
                            : (const void*)&detail::k_w4_split<kX, kW, kS, kMode, 2, 4>;
      case 3: return nt == 2 ? (const void*)&detail::k_w4_split<kX, kW, kS, kMode, 3, 2>
                            : (const void*)&detail::k_w4_split<kX, kW, kS, kMode, 3, 4>;
      default: return nt == 2 ? (const void*)&detail::k_w4_split<kX, kW, kS, kMode, 4, 2>
                            : (const void*)&detail::k_w4_split<kX, kW, kS, kMode, 4, 4>;
    }
  });
}

template <int kX, int kW>
const void* moe_up_of(int s, int mode, int mt, int wk) {
  return sel_scales<kX, kW>(s, mode, [&](auto S, auto Mode) {
    return sel_mt(mt, [&](auto MT) {
      constexpr int kS = decltype(S)::value, kMode = decltype(Mode)::value;
      constexpr int kMT = decltype(MT)::value;
      return wk == 8 ? (const void*)&detail::k_moe_up<kX, kW, kS, kMode, kMT, 8>
                     : (const void*)&detail::k_moe_up<kX, kW, kS, kMode, kMT, 2>;
    });
  });
}

// Scale types as above, whatever the mode.
template <int kW, class F>
const void* sel_vec(int s, int lk, F&& f) {
  using namespace detail;
  auto by_lk = [&](auto S) { return lk == 64 ? f(S, ic<64>{}) : f(S, ic<16>{}); };
  if constexpr (kW == kWE4M3) return s == kInF32 ? by_lk(ic<kInF32>{}) : nullptr;
  else return sel4(s, by_lk);
}
template <int kX, int kW>
const void* moe_vec_up_of(int s, int lk) {
  return sel_vec<kW>(s, lk, [](auto S, auto L) {
    return (const void*)&detail::k_moe_vec_up<kX, kW, decltype(S)::value, decltype(L)::value>;
  });
}
template <int kW>
const void* moe_vec_down_of(int s, int lk, int h) {
  return sel_vec<kW>(s, lk, [h](auto S, auto L) {
    constexpr int kS = decltype(S)::value, kLk = decltype(L)::value;
    return h == 3 ? (const void*)&detail::k_moe_vec_down<kW, kS, kLk, 3>
                  : (const void*)&detail::k_moe_vec_down<kW, kS, kLk, 2>;
  });
}

// h: parts of h; tiles of three are of 16 rows.
template <int kW>
const void* moe_down_of(int s, int mode, int mt, int wk, int h) {
  return sel_scales<detail::kInBf16, kW>(s, mode, [&](auto S, auto Mode) -> const void* {
    constexpr int kS = decltype(S)::value, kMode = decltype(Mode)::value;
    if (h == 3)
      return mt != 1 ? nullptr
             : wk == 8 ? (const void*)&detail::k_moe_down<kW, kS, kMode, 1, 8, 3>
                       : (const void*)&detail::k_moe_down<kW, kS, kMode, 1, 2, 3>;
    return sel_mt(mt, [&](auto MT) {
      constexpr int kMT = decltype(MT)::value;
      return wk == 8 ? (const void*)&detail::k_moe_down<kW, kS, kMode, kMT, 8, 2>
                     : (const void*)&detail::k_moe_down<kW, kS, kMode, kMT, 2, 2>;
    });
  });
}

}  // namespace kernels
}  // namespace hipgemm
