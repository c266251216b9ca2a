// The paged grouped-head attention kernels for f16 tensors.
#include "paged_gqa.h"

namespace mls {
template int gqa_launch<_Float16>(const GqaArgs&, const GqaShape&, int64_t, hipStream_t);
template void gqa_tiles<_Float16>(GqaShape&);
}  // namespace mls
