// Group norm kernels over bf16 maps (group_norm.h).
#include "group_norm.h"

namespace gn {
int launch_bf16(const Plan& p, const Args& a, hipStream_t st) { return launch<bf16>(p, a, st); }
}  // namespace gn
