// Dispatch of the residual-stream kernels by element type (residual.cuh).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "residual.h"

namespace cfb {

template <typename T>
int join_fwd_t(const JoinArgs& a, int num_sms, cudaStream_t s);
template <typename T>
int join_bwd_blocks_t(const JoinArgs& a, int num_sms);
template <typename T>
int join_bwd_t(const JoinArgs& a, int num_sms, cudaStream_t s);
template <typename T>
int dropout_t(const void* x, void* y, int64_t n, const DropArgs& d, cudaStream_t s);

bool join_width_ok(int H) { return H <= (H % 8 == 0 ? kJoinMaxWidth : kJoinMaxOdd); }

int join_fwd(const JoinArgs& a, int num_sms, cudaStream_t s) {
  if (a.T == 0) return 0;
  return a.type == kStreamBf16   ? join_fwd_t<__nv_bfloat16>(a, num_sms, s)
         : a.type == kStreamHalf ? join_fwd_t<__half>(a, num_sms, s)
                                 : join_fwd_t<float>(a, num_sms, s);
}

int join_bwd_blocks(const JoinArgs& a, int num_sms) {
  return a.type == kStreamBf16   ? join_bwd_blocks_t<__nv_bfloat16>(a, num_sms)
         : a.type == kStreamHalf ? join_bwd_blocks_t<__half>(a, num_sms)
                                 : join_bwd_blocks_t<float>(a, num_sms);
}

int join_bwd(const JoinArgs& a, int num_sms, cudaStream_t s) {
  return a.type == kStreamBf16   ? join_bwd_t<__nv_bfloat16>(a, num_sms, s)
         : a.type == kStreamHalf ? join_bwd_t<__half>(a, num_sms, s)
                                 : join_bwd_t<float>(a, num_sms, s);
}

int dropout_run(const void* x, void* y, int64_t n, int type, const DropArgs& d, cudaStream_t s) {
  if (n == 0) return 0;
  return type == kStreamBf16   ? dropout_t<__nv_bfloat16>(x, y, n, d, s)
         : type == kStreamHalf ? dropout_t<__half>(x, y, n, d, s)
                               : dropout_t<float>(x, y, n, d, s);
}

}  // namespace cfb
