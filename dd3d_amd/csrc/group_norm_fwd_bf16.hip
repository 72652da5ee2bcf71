// The group norm's forward pass for bf16 rows (group_norm.h).
#include "group_norm_launch.h"

namespace gn {
template int launch_fwd<bf16_t>(const Norm&, const Plan&, const void*, void*, float*, float*, const Work&, hipStream_t);
}  // namespace gn
