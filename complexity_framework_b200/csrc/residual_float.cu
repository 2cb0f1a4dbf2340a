// The residual-stream kernels of float tensors.
#include "residual.cuh"

namespace cfb {
CFB_STREAM_TYPE(float)
}  // namespace cfb
