// Host interface of the cross-entropy over the vocabulary (vocab_loss.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace cfb {

// Rows of the compact copies: the counted rows in their order, then zero rows up to a whole
// 64-row block (the K step of the weight gradient).
inline int64_t vl_rows(int64_t T) { return T <= 64 ? 64 : (T + 63) / 64 * 64; }

// One call.  Index tensors, with R = vl_rows(T):
//   cnt    [2]  counted rows, and the same but at least 1 (rows that the products take)
//   target [R]  word of each compact row, -1: none        src [R]  its row in the call, -1: none
//   pos    [T]  compact row of each row, -1: not counted
struct VlCall {
  int64_t T = 0;
  int V = 0, H = 0;
  float scale = 1.f, smooth = 0.f, z = 0.f;
  float sign = 1.f;                  // of the row losses (-1: log-probabilities)
  int64_t ignore = -100;
  const __nv_bfloat16* w = nullptr;  // [V, H]
  __nv_bfloat16* hc = nullptr;       // [R, H] compact rows
  int *cnt = nullptr, *target = nullptr, *src = nullptr, *pos = nullptr;
  float* lse2 = nullptr;             // [R] log-sum-exp of each compact row, in units of log 2
  float* ginv = nullptr;             // [1] factor of the loss's sum
  int num_sms = 148;
  int* err = nullptr;
};

struct VlForward {
  const __nv_bfloat16* h = nullptr;  // [T, H]
  const int64_t* targets = nullptr;  // [T]
  float* rows = nullptr;             // [T] loss of each row
  float* total = nullptr;            // [1] or null: ginv times their sum
  bool mean = false;                 // ginv = 1 / counted rows, else 1
  float* ws = nullptr;               // vl_forward_floats
};
int64_t vl_forward_floats(const VlCall& c);
int vl_forward(const VlCall& c, const VlForward& f, cudaStream_t s);

struct VlBackward {
  const float* gout = nullptr;       // [1], or [T] with per_row
  bool per_row = false;
  __nv_bfloat16* dh = nullptr;       // [T, H] or null
  __nv_bfloat16* dw = nullptr;       // [V, H] or null
  // plan: words a piece, K slices of the hidden gradient
  int piece = 0, ksplit = 1;
  __nv_bfloat16* dl = nullptr;       // [R, piece]
  float* acc = nullptr;              // vl_acc_floats
  float* resid = nullptr;            // [R] what rounding took from each row's target
  float* alpha = nullptr;            // [1] workspace: the factor that all rows share
};
void vl_backward_plan(const VlCall& c, int64_t workspace_bytes, VlBackward* b);
int64_t vl_acc_floats(const VlCall& c, const VlBackward& b);
int vl_backward(const VlCall& c, const VlBackward& b, cudaStream_t s);

}  // namespace cfb
