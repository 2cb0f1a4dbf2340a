// The residual-stream kernels of __nv_bfloat16 tensors.
#include "residual.cuh"

namespace cfb {
CFB_STREAM_TYPE(__nv_bfloat16)
}  // namespace cfb
