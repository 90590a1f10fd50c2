// Products of bf16 operands: both operands along K, with a residual.
#include "kdense.hpp"

namespace hipgemm {
namespace kernels {

const void* dense_tile_bf16_res(int tile, int mode) {
  return dense_tile_of<detail::kInBf16, false, false, detail::kEpiResidual>(tile, mode);
}

}  // namespace kernels
}  // namespace hipgemm
