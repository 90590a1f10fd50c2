// Products of bf16 operands: both operands across K.
#include "kdense.hpp"

namespace hipgemm {
namespace kernels {

const void* dense_tile_bf16_tn(int tile, int mode) {
  return dense_tile_of<detail::kInBf16, true, true, detail::kEpiPlain>(tile, mode);
}

}  // namespace kernels
}  // namespace hipgemm
