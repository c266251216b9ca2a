// The paged grouped-head attention kernels for bf16 tensors.
#include "paged_gqa.h"

namespace mls {
template int gqa_launch<__bf16>(const GqaArgs&, const GqaShape&, int64_t, hipStream_t);
template void gqa_tiles<__bf16>(GqaShape&);
}  // namespace mls
