// Products of f16 operands: the second operand across K.
#include "kdense.hpp"

namespace hipgemm {
namespace kernels {

const void* dense_tile_f16_nn(int tile, int mode) {
  return dense_tile_of<detail::kInF16, false, true, detail::kEpiPlain>(tile, mode);
}

}  // namespace kernels
}  // namespace hipgemm
