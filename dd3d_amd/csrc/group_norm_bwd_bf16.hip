// The group norm's first gradient for bf16 rows (group_norm.h).
#include "group_norm_launch.h"

namespace gn {
template int launch_bwd<bf16_t>(const Norm&, const Plan&, const void*, const void*, const float*, const float*, void*, const Work&, Fold, hipStream_t);
}  // namespace gn
