#include "fg_mx_kernels.h"

namespace fg {

hipError_t launch_mx_attn_fp16(const MxAttnArgs& m, hipStream_t st) { return launch_mx_items<false>(m, st); }

}  // namespace fg
