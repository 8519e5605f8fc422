// The attention kernels for fp16 queries.
#include "fg_attn_kernels.h"

namespace fg {
hipError_t launch_attn_fp16(const AttnArgs& a, bool fp8, int kind, hipStream_t st) {
  return launch_attn_items<false>(a, fp8, kind, st);
}
}  // namespace fg
