// The attention kernels for bf16 queries.
#include "fg_attn_kernels.h"

namespace fg {
hipError_t launch_attn_bf16(const AttnArgs& a, bool fp8, int kind, hipStream_t st) {
  return launch_attn_items<true>(a, fp8, kind, st);
}
}  // namespace fg
