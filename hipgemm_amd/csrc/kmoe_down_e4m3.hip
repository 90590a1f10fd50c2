// The experts' down products with e4m3 weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_down_e4m3(int s, int mode, int mt, int wk) {
  return moe_down_of<detail::kWE4M3>(s, mode, mt, wk);
}
const void* moe_vec_down_e4m3(int s, int lk) {
  return moe_vec_down_of<detail::kWE4M3>(s, lk);
}

}  // namespace kernels
}  // namespace hipgemm
