// Products of bf16 operands: both operands across K.
#include "kdense.hpp"

namespace hipgemm {
namespace kernels {

const void* dense_tile_bf16_tn(int tile, bool split) {
  return dense_tile_of<detail::kInBf16, true, true, detail::kEpiPlain>(tile, split);
}

}  // namespace kernels
}  // namespace hipgemm
