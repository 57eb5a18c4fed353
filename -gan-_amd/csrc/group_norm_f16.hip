// Group norm kernels over f16 maps (group_norm.h).
#include "group_norm.h"

namespace gn {
int launch_f16(const Plan& p, const Args& a, hipStream_t st) { return launch<f16>(p, a, st); }
}  // namespace gn
