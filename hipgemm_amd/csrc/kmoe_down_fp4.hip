// The experts' down products with fp4 weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_down_fp4(int s, int mode, int mt, int wk) {
  return moe_down_of<detail::kWFp4>(s, mode, mt, wk);
}
const void* moe_vec_down_fp4(int s, int lk) {
  return moe_vec_down_of<detail::kWFp4>(s, lk);
}

}  // namespace kernels
}  // namespace hipgemm
