// The experts' products with e4m3 weights.
#include "kmoe.hpp"

namespace hipgemm {
namespace kernels {

const void* moe_up_e4m3(int x, int s, int mode, int mt) {
  return x == detail::kInBf16 ? moe_up_of<detail::kInBf16, detail::kWE4M3>(s, mode, mt)
                              : moe_up_of<detail::kInF16, detail::kWE4M3>(s, mode, mt);
}
const void* moe_down_e4m3(int s, int mode) { return moe_down_of<detail::kWE4M3>(s, mode); }

}  // namespace kernels
}  // namespace hipgemm
