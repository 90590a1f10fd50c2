// The experts' down products with fp4 weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_down_fp4(int s, int mode, int mt, int wk, int h) {
  return moe_down_of<detail::kWFp4>(s, mode, mt, wk, h);
}
const void* moe_vec_down_fp4(int s, int lk, int h) {
  return moe_vec_down_of<detail::kWFp4>(s, lk, h);
}

}  // namespace kernels
}  // namespace hipgemm
