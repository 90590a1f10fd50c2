// Products of f16 operands: both operands along K, bias and activation.
#include "kdense.hpp"

namespace hipgemm {
namespace kernels {

const void* dense_tile_f16_nt(int tile, int mode) {
  return dense_tile_of<detail::kInF16, false, false, detail::kEpiLinear>(tile, mode);
}

}  // namespace kernels
}  // namespace hipgemm
