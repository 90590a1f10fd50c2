// The experts' gate and up products, f16 activations, int4z weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_up_f16_int4z(int s, int mode, int mt, int wk) {
  return moe_up_of<detail::kInF16, detail::kWInt4Z>(s, mode, mt, wk);
}
const void* moe_vec_up_f16_int4z(int s, int lk) {
  return moe_vec_up_of<detail::kInF16, detail::kWInt4Z>(s, lk);
}

}  // namespace kernels
}  // namespace hipgemm
