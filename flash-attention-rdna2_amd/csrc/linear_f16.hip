// Linear attention kernels for _Float16 (see linear_kernel.hpp).
#include "linear_kernel.hpp"

namespace fa {
template <>
int la_launch<_Float16>(const LaArgs& p, bool state, hipStream_t st) {
  return state ? la_pick<_Float16, true>(p, st) : la_pick<_Float16, false>(p, st);
}
}  // namespace fa
