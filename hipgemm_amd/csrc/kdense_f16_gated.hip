// Products of f16 operands: gate and up rows.
#include "kdense.hpp"

namespace hipgemm {
namespace kernels {

const void* dense_tile_f16_gated(int tile, int mode) {
  return dense_tile_of<detail::kInF16, false, false, detail::kEpiGated>(tile, mode);
}

}  // namespace kernels
}  // namespace hipgemm
