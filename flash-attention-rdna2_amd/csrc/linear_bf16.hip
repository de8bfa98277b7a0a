// Linear attention kernels for __bf16.
#include "linear_kernel.hpp"

namespace fa {
template <>
void la_launch<__bf16>(const LaPasses& p, bool state, bool exact, hipStream_t st) {
  exact ? la_all<__bf16, 3>(p, state, st) : la_all<__bf16, 2>(p, state, st);
}
}  // namespace fa
