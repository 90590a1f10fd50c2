// Products of bf16 operands: gate and up rows.
#include "kdense.hpp"

namespace hipgemm {
namespace kernels {

const void* dense_tile_bf16_gated(int tile, int mode) {
  return dense_tile_of<detail::kInBf16, false, false, detail::kEpiGated>(tile, mode);
}

}  // namespace kernels
}  // namespace hipgemm
