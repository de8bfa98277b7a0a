// Linear attention kernels for float.
#include "linear_kernel.hpp"

namespace fa {
template <>
void la_launch<float>(const LaPasses& p, bool state, bool, hipStream_t st) {
  la_all<float, 1>(p, state, st);
}
}  // namespace fa
