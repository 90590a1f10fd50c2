// The experts' down products with e4m3 weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_down_e4m3(int s, int mode, int mt, int wk, int h) {
  return moe_down_of<detail::kWE4M3>(s, mode, mt, wk, h);
}
const void* moe_vec_down_e4m3(int s, int lk, int h) {
  return moe_vec_down_of<detail::kWE4M3>(s, lk, h);
}

}  // namespace kernels
}  // namespace hipgemm
