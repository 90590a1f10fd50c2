// Instantiations of the products of 16-bit operands (dense.hpp): one file per operand
// type and layout.
#pragma once

#include "kernels.hpp"

#include "hipgemm/detail/dense.hpp"

namespace hipgemm {
namespace kernels {

template <class Cfg, int kX, bool kACol, bool kBCol, int kEpi, bool kSplit, bool kOnce>
__global__ __launch_bounds__(256, 1) void k_dense_tile(detail::DenseArgs g) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsBytes];
  detail::dense_tile_body<Cfg, kX, kACol, kBCol, kEpi, kSplit, kOnce>(
      g, (detail::lds_u8*)lds, blockIdx.x, gridDim.x);
}

// The two products of a backward pass, in tiles that have a CU each: half of the chip is all
// that either takes (1531 x 2001 x 1000: 18 and 17 us one after the other, 24 together).
template <int kX>
__global__ __launch_bounds__(256, 1) void k_dense_tile_pair(detail::DensePair g) {
  using Cfg = detail::CfgDense<kDenseTiles[0].bm, kDenseTiles[0].bn, 4>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsBytes];
  const int b = blockIdx.x;
  if (b < g.first)
    detail::dense_tile_body<Cfg, kX, false, true, detail::kEpiPlain, false>(
        g.x, (detail::lds_u8*)lds, b, g.first);
  else
    detail::dense_tile_body<Cfg, kX, true, true, detail::kEpiPlain, false>(
        g.w, (detail::lds_u8*)lds, b - g.first, gridDim.x - g.first);
}

template <class Cfg, int kX, bool kACol, bool kBCol, int kEpi>
const void* dense_tile_mode(int mode) {
  // (Sums in slices know of the gate only.)
  constexpr int kPart = kEpi == detail::kEpiGated ? kEpi : detail::kEpiPlain;
  constexpr bool kOnce = Cfg::kBM == 64 && !kBCol;
  switch (mode) {
    case 0: return (const void*)&k_dense_tile<Cfg, kX, kACol, kBCol, kEpi, false, false>;
    case kDenseSplit:
      return (const void*)&k_dense_tile<Cfg, kX, kACol, kBCol, kPart, true, false>;
    case kDenseOnce:
      if constexpr (kOnce)
        return (const void*)&k_dense_tile<Cfg, kX, kACol, kBCol, kEpi, false, true>;
      return nullptr;
    default:
      if constexpr (kOnce)
        return (const void*)&k_dense_tile<Cfg, kX, kACol, kBCol, kPart, true, true>;
      return nullptr;
  }
}

// tile: index of kDenseTiles.
template <int kX, bool kACol, bool kBCol, int kEpi>
const void* dense_tile_of(int tile, int mode) {
  using namespace detail;
  auto of = [&](auto cfg) {
    return dense_tile_mode<decltype(cfg), kX, kACol, kBCol, kEpi>(mode);
  };
  switch (tile) {
    case 0: return of(CfgDense<kDenseTiles[0].bm, kDenseTiles[0].bn, 4>{});
    case 1: return of(CfgDense<kDenseTiles[1].bm, kDenseTiles[1].bn, 2>{});
    case 2: return kACol ? nullptr : of(CfgDense<kDenseTiles[2].bm, kDenseTiles[2].bn, 6>{});
    case 3: return of(CfgDense<kDenseTiles[3].bm, kDenseTiles[3].bn, 3>{});
    default: return nullptr;
  }
}

}  // namespace kernels
}  // namespace hipgemm
