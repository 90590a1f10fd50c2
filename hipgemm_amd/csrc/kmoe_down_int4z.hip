// The experts' down products with int4z weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_down_int4z(int s, int mode, int mt, int wk) {
  return moe_down_of<detail::kWInt4Z>(s, mode, mt, wk);
}
const void* moe_vec_down_int4z(int s, int lk) {
  return moe_vec_down_of<detail::kWInt4Z>(s, lk);
}

}  // namespace kernels
}  // namespace hipgemm
