// Products of bf16 operands: both operands along K, bias and activation.
#include "kdense.hpp"

namespace hipgemm {
namespace kernels {

const void* dense_tile_bf16_nt(int tile, int mode) {
  return dense_tile_of<detail::kInBf16, false, false, detail::kEpiLinear>(tile, mode);
}

}  // namespace kernels
}  // namespace hipgemm
