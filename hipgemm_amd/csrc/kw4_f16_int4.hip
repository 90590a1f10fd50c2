// Products of f16 activations with int4 weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* w4_vec_f16_int4(int s, int rows, int lk) {
  return w4_vec_of<detail::kInF16, detail::kWInt4>(s, rows, lk);
}
const void* w4_tile_f16_int4(int s, int mode) {
  return w4_tile_of<detail::kInF16, detail::kWInt4>(s, mode);
}
const void* w4_split_f16_int4(int s, int mode, int mt, int nt) {
  return w4_split_of<detail::kInF16, detail::kWInt4>(s, mode, mt, nt);
}

}  // namespace kernels
}  // namespace hipgemm
