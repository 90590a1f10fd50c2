// Products of bf16 operands: the second operand across K; a backward pass' two
// products together.
#include "kdense.hpp"

namespace hipgemm {
namespace kernels {

const void* dense_tile_bf16_nn(int tile, int mode) {
  return dense_tile_of<detail::kInBf16, false, true, detail::kEpiPlain>(tile, mode);
}
const void* dense_pair_bf16() { return (const void*)&k_dense_tile_pair<detail::kInBf16>; }

}  // namespace kernels
}  // namespace hipgemm
