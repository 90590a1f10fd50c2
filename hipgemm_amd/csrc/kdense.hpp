// Instantiations of the products of 16-bit operands (dense.hpp): one file per operand
// type and layout.
#pragma once

#include "kernels.hpp"

#include "hipgemm/detail/dense.hpp"

namespace hipgemm {
namespace kernels {

template <class Cfg, int kX, bool kACol, bool kBCol, int kEpi, bool kSplit>
__global__ __launch_bounds__(256, 1) void k_dense_tile(detail::DenseArgs g) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsBytes];
  detail::dense_tile_body<Cfg, kX, kACol, kBCol, kEpi, kSplit>(g, (detail::lds_u8*)lds);
}

// tile: index of kDenseTiles.
template <int kX, bool kACol, bool kBCol, int kEpi>
const void* dense_tile_of(int tile, bool split) {
  auto of = [&](auto cfg) {
    return sel2(split, [&](auto s) {
      return (const void*)&k_dense_tile<decltype(cfg), kX, kACol, kBCol, kEpi,
                                        decltype(s)::value>;
    });
  };
  switch (tile) {
    case 0: return of(detail::CfgDense<kDenseTiles[0].bm, kDenseTiles[0].bn, 4>{});
    case 1: return of(detail::CfgDense<kDenseTiles[1].bm, kDenseTiles[1].bn, 2>{});
    default: return nullptr;
  }
}

}  // namespace kernels
}  // namespace hipgemm
