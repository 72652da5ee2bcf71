// The group norm's second gradient for bf16 rows (group_norm.h).
#include "group_norm_launch.h"

namespace gn {
template int launch_bwd2<bf16_t>(const Norm&, const Plan&, const void*, const void*, const void*, const void*, const void*, const float*, const float*, void*, void*, const Work&, Fold, hipStream_t);
}  // namespace gn
