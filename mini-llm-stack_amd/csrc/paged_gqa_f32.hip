// The paged grouped-head attention kernels for f32 tensors.
#include "paged_gqa.h"

namespace mls {
template int gqa_launch<float>(const GqaArgs&, const GqaShape&, int64_t, hipStream_t);
template void gqa_tiles<float>(GqaShape&);
}  // namespace mls
