// Host interface of the residual-stream kernels (residual.cuh).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace cfb {

enum StreamType : int { kStreamBf16 = 0, kStreamHalf = 1, kStreamFloat = 2 };

// The counter-based generator of one dropout call: kept where 16 random bits >= threshold.
struct DropArgs {
  const int64_t* seed_ptr = nullptr;  // device seed, or null for `seed`
  uint64_t seed = 0;
  uint32_t stream = 0;
  int threshold = 0;  // round(p * 65536); 0 = no dropout
  float factor() const { return threshold >= 65536 ? 0.f : 65536.f / (65536 - threshold); }
};

// x' = x + scale * drop(gate * w1 * b / rms(b)),  y = w2 * x' / rms(x').
// w1, gate and w2 may be null (no norm, no gate, no y).
struct JoinArgs {
  const void *x = nullptr, *b = nullptr, *w1 = nullptr, *gate = nullptr, *w2 = nullptr;
  void *xnew = nullptr, *y = nullptr;   // forward: outputs; backward: xnew is the saved x'
  float *r1 = nullptr, *r2 = nullptr;   // 1 / rms of each row (written forward unless null)
  const void *dxnew = nullptr, *dy = nullptr;        // backward inputs, either may be null
  void *dx = nullptr, *db = nullptr;                 // backward outputs, either may be null
  void *dw1 = nullptr, *dgate = nullptr, *dw2 = nullptr;  // may be null
  float* partials = nullptr;                         // [join_bwd_blocks][2][H]
  DropArgs drop;
  float scale = 1.f, eps = 1e-6f;
  int64_t T = 0;
  int H = 0;
  int type = kStreamBf16;
  int* err = nullptr;                                // device error word
};

// Widest rows: 2048 blocks of eight elements, of which the ends of odd rows take one more.
constexpr int kJoinMaxWidth = 16384, kJoinMaxOdd = 16370;

bool join_width_ok(int H);
int join_fwd(const JoinArgs& a, int num_sms, cudaStream_t s);
int join_bwd_blocks(const JoinArgs& a, int num_sms);
int join_bwd(const JoinArgs& a, int num_sms, cudaStream_t s);
int dropout_run(const void* x, void* y, int64_t n, int type, const DropArgs& d, cudaStream_t s);

}  // namespace cfb
