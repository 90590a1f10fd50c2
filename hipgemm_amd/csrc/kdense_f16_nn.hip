// Products of f16 operands: the second operand across K; a backward pass' two
// products together.
#include "kdense.hpp"

namespace hipgemm {
namespace kernels {

const void* dense_tile_f16_nn(int tile, int mode) {
  return dense_tile_of<detail::kInF16, false, true, detail::kEpiPlain>(tile, mode);
}
const void* dense_pair_f16() { return (const void*)&k_dense_tile_pair<detail::kInF16>; }

}  // namespace kernels
}  // namespace hipgemm
