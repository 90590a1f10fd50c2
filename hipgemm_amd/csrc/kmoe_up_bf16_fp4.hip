// The experts' gate and up products, bf16 activations, fp4 weights.
#include "kw4.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_up_bf16_fp4(int s, int mode, int mt, int wk) {
  return moe_up_of<detail::kInBf16, detail::kWFp4>(s, mode, mt, wk);
}
const void* moe_vec_up_bf16_fp4(int s, int lk) {
  return moe_vec_up_of<detail::kInBf16, detail::kWFp4>(s, lk);
}

}  // namespace kernels
}  // namespace hipgemm
