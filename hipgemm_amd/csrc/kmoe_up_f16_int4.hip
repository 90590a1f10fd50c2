// The experts' gate and up products, f16 activations, int4 weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_up_f16_int4(int s, int mode, int mt, int wk) {
  return moe_up_of<detail::kInF16, detail::kWInt4>(s, mode, mt, wk);
}
const void* moe_vec_up_f16_int4(int s, int lk) {
  return moe_vec_up_of<detail::kInF16, detail::kWInt4>(s, lk);
}

}  // namespace kernels
}  // namespace hipgemm
