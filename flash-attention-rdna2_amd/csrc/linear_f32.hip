// Linear attention kernels for float (see linear_kernel.hpp).
#include "linear_kernel.hpp"

namespace fa {
template <>
int la_launch<float>(const LaArgs& p, bool state, hipStream_t st) {
  return state ? la_pick<float, true>(p, st) : la_pick<float, false>(p, st);
}
}  // namespace fa
