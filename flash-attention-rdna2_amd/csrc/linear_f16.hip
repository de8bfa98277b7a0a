// Linear attention kernels for _Float16.
#include "linear_kernel.hpp"

namespace fa {
template <>
void la_launch<_Float16>(const LaPasses& p, bool state, bool exact, hipStream_t st) {
  exact ? la_all<_Float16, 3>(p, state, st) : la_all<_Float16, 2>(p, state, st);
}
}  // namespace fa
