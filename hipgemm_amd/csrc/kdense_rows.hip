// Products of a few rows of 16-bit operands (dense_rows.hpp).
#include "kernels.hpp"

#include "hipgemm/detail/dense_rows.hpp"

namespace hipgemm {
namespace kernels {
namespace {

using namespace detail;

template <int kX, int kMT, int kEpi>
__global__ __launch_bounds__(256, 2) void k_dense_rows(DenseArgs g) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[CfgRows<kMT>::kLdsBytes];
  dense_rows_body<kX, kMT, kEpi>(g, (lds_u8*)lds);
}

template <int kX, int kMT>
const void* rows_of(int kind) {
  switch (kind) {
    case kDenseNT: return (const void*)&k_dense_rows<kX, kMT, kEpiLinear>;
    case kDenseRes: return (const void*)&k_dense_rows<kX, kMT, kEpiResidual>;
    case kDenseGated: return (const void*)&k_dense_rows<kX, kMT, kEpiGated>;
    default: return nullptr;
  }
}

}  // namespace

const void* dense_rows(int x, int kind, int mt) {
  return sel2(x == kInBf16, [&](auto b) {
    constexpr int kX = decltype(b)::value ? kInBf16 : kInF16;
    return mt == 1 ? rows_of<kX, 1>(kind) : mt == 2 ? rows_of<kX, 2>(kind)
                                                    : rows_of<kX, 4>(kind);
  });
}

}  // namespace kernels
}  // namespace hipgemm
