// The residual-stream kernels of __half tensors.
#include "residual.cuh"

namespace cfb {
CFB_STREAM_TYPE(__half)
}  // namespace cfb
