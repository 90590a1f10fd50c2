// Products of bf16 activations with int4 weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* w4_vec_bf16_int4(int s, int rows, int lk) {
  return w4_vec_of<detail::kInBf16, detail::kWInt4>(s, rows, lk);
}
const void* w4_rows_bf16_int4(int s, int mode, int mt) {
  return w4_rows_of<detail::kInBf16, detail::kWInt4>(s, mode, mt);
}

}  // namespace kernels
}  // namespace hipgemm
