// Group norm kernels over f32 maps (group_norm.h).
#include "group_norm.h"

namespace gn {
int launch_f32(const Plan& p, const Args& a, hipStream_t st) { return launch<float>(p, a, st); }
}  // namespace gn
