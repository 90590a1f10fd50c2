// The experts' products with fp4 weights.
#include "kmoe.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_up_fp4(int x, int s, int mode, int mt) {
  return x == detail::kInBf16 ? moe_up_of<detail::kInBf16, detail::kWFp4>(s, mode, mt)
                              : moe_up_of<detail::kInF16, detail::kWFp4>(s, mode, mt);
}
const void* moe_down_fp4(int s, int mode) { return moe_down_of<detail::kWFp4>(s, mode); }

}  // namespace kernels
}  // namespace hipgemm
