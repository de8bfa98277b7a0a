// Linear attention kernels for __bf16 (see linear_kernel.hpp).
#include "linear_kernel.hpp"

namespace fa {
template <>
int la_launch<__bf16>(const LaArgs& p, bool state, hipStream_t st) {
  return state ? la_pick<__bf16, true>(p, st) : la_pick<__bf16, false>(p, st);
}
}  // namespace fa
