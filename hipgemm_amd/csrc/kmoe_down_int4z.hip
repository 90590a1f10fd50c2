// The experts' down products with int4z weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_down_int4z(int s, int mode, int mt, int wk, int h) {
  return moe_down_of<detail::kWInt4Z>(s, mode, mt, wk, h);
}
const void* moe_vec_down_int4z(int s, int lk, int h) {
  return moe_vec_down_of<detail::kWInt4Z>(s, lk, h);
}

}  // namespace kernels
}  // namespace hipgemm
