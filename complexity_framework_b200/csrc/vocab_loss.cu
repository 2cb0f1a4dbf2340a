// Softmax cross-entropy over a large vocabulary, and its gradients, without keeping the logits.
//
// With z_v = scale * h . w_v, lse = log sum_v exp(z_v) and p_v = exp(z_v - lse), a counted row
// with the word y has
//
//   loss = lse - (1 - eps) z_y - eps / V sum_v z_v + lambda lse^2
//   d loss / d z_v = p_v (1 + 2 lambda lse) - (1 - eps) [v = y] - eps / V
//
// Forward: one product h W^T whose epilogue leaves, of each row's 128 words, their maximum, the
// sum of exponentials and (for smoothing) the sum, and the target's logit: 1/16 of a bf16 logit
// matrix's bytes.  Backward: for a piece of the vocabulary at a time, the product again with an
// epilogue that writes d loss / d z in bf16, then dh += dz W and dW = dz^T h.  That is four
// products of 2 T V H operations where three would do with the logits kept; all run on the
// tensor cores from fp32 accumulators, and the logits are never rounded to bf16.
//
// The products of 8192 x 32000 x 896, ncu at the 1.46 GHz of the power limit: logits 289 us
// with the tensor pipe active 92 % of the time, dz 328 us (79 %), dh 356 (75 %), dW 335 (79 %).  A
// whole call with gradients: 32768 x 32000 x 896 in 7.0 ms, 4096 x 100000 x 4096 in 10.4 ms (1.1
// and 1.3 PFLOP/s of the four products; cuBLAS runs 1.41 back to back).
//
// Rows that do not count (ignored targets) are left out before the first product: the others are
// gathered in their order, and the products take their number from device memory.  A batch with
// half of its tokens ignored costs half, and what an ignored row holds reaches nothing.
//
// dz is rounded to bf16, as the tensor cores' operand (gradients are off by up to 0.0024, root mean
// square, where their own rounding gives 0.0017); its sums are fp32.  The factors that all
// rows share (1 / counted rows, the incoming gradient, scale, 1 - eps) are left to the products'
// epilogues, so that a target's term is p - 1 and the -1 is exact: scaled first, every target's
// term would be off by the same part of up to 2^-9.  What rounding the target's term takes is put back
// into dh (vl_scatter_k); in dW, a sum over rows with errors of either sign, it stays.  The
// exponentials are ex2.approx's (2^-22): row losses are off by 3.4e-7 of their size where fp32
// elementary operations give 1.3e-7.  No sum depends on the order of atomics: equal calls give
// equal bits.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "gemm_tc.h"
#include "vocab_loss.h"

namespace cfb {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The counted rows in their order: every block of `per` rows counts the rows before its own, so
// one launch does, without atomics.  At most 4 blocks an SM read targets (592 on 148 SMs, on average
// half of them: 2.4 KB a row, from L2), so that the reads grow with the rows.
__global__ void __launch_bounds__(256) vl_gather_k(const VlCall c, const VlForward f, int per) {
  __shared__ int warp_n[8];
  __shared__ int dest[256];
  grid_dependents_go();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nv = c.H >> 3;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per;
  const auto counts = [&](int64_t y) { return y != c.ignore && y >= 0 && y < c.V; };
  int before = 0;
  int64_t i0 = tid;
  for (; i0 + 7 * 256 < first; i0 += 8 * 256) {  // eight loads under way
    int64_t v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = f.targets[i0 + k * 256];
#pragma unroll
    for (int k = 0; k < 8; ++k) before += counts(v[k]) ? 1 : 0;
  }
  for (; i0 < first; i0 += 256) before += counts(f.targets[i0]) ? 1 : 0;
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) warp_n[warp] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) before += warp_n[k];
  __syncthreads();
  const int64_t last = first + per < c.T ? first + per : c.T;
  int end = before;
  for (int64_t r0 = first; r0 < last; r0 += 256) {  // 256 rows at a time
    before = end;
    const int rows = last - r0 < 256 ? static_cast<int>(last - r0) : 256;
    const int64_t row = r0 + tid;
    const bool mine = tid < rows;
    const int64_t y = mine ? f.targets[row] : c.ignore;
    const bool on = mine && counts(y);
    const uint32_t ballot = __ballot_sync(0xffffffffu, on);
    if (lane == 0) warp_n[warp] = __popc(ballot);
    __syncthreads();
    int at = before;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k < warp) at += warp_n[k];
      end += warp_n[k];
    }
    at += __popc(ballot & ((1u << lane) - 1u));
    if (mine) {
      dest[tid] = on ? at : -1;
      c.pos[row] = on ? at : -1;
      if (on) {
        c.target[at] = static_cast<int>(y);
        c.src[at] = static_cast<int>(row);
      } else {
        // a target that is neither a word nor ignored: reported, and a loss of NaN
        if (y != c.ignore) report_error(c.err, kErrBounds, 60);
        f.rows[row] = y == c.ignore ? 0.f : NAN;
      }
    }
    __syncthreads();
    for (int q0 = warp; q0 < rows; q0 += 4 * 8) {  // four rows a warp at a time
      const uint4* in[4];
      uint4* out[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int q = q0 + k * 8;
        const int to = q < rows ? dest[q] : -1;
        in[k] = to < 0 ? nullptr : reinterpret_cast<const uint4*>(f.h + (r0 + q) * c.H);
        out[k] = to < 0 ? nullptr
                        : reinterpret_cast<uint4*>(c.hc + static_cast<int64_t>(to) * c.H);
      }
#pragma unroll 2
      for (int i = lane; i < nv; i += 32) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (in[k] != nullptr) v[k] = in[k][i];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (in[k] != nullptr) out[k][i] = v[k];
      }
    }
  }
  if (blockIdx.x + 1 < gridDim.x) return;
  // the last block knows the count; rows up to the next whole block of 64 become 0
  const int64_t stop = end <= 64 ? 64 : (static_cast<int64_t>(end) + 63) / 64 * 64;
  for (int64_t r = end + warp; r < stop; r += 8) {
    uint4* out = reinterpret_cast<uint4*>(c.hc + r * c.H);
    for (int i = lane; i < nv; i += 32) out[i] = make_uint4(0u, 0u, 0u, 0u);
    if (lane == 0) {
      c.target[r] = -1;
      c.src[r] = -1;
    }
  }
  if (tid == 0) {
    c.cnt[0] = end;
    c.cnt[1] = end > 0 ? end : 1;
    *c.ginv = f.mean ? 1.f / static_cast<float>(end > 0 ? end : 1) : 1.f;
  }
}

// Joins the half tiles' statistics of rows [first, first + n), a warp a row.
__global__ void __launch_bounds__(256) vl_rows_k(const VlCall c, const VlForward f,
                                                 const float2* stats, const float* zt,
                                                 const float* zsum, int halves, int64_t first,
                                                 int64_t n) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t row = first + at;
  if (at >= n || row >= c.cnt[1]) return;
  const float2* st = stats + at * halves;
  float mx = -INFINITY;
  for (int i = lane; i < halves; i += 32) mx = fmaxf(mx, st[i].x);
  mx = warp_max(mx);
  const float k2 = c.scale * kLog2e;
  float se = 0.f, zs = 0.f;
  for (int i = lane; i < halves; i += 32) {
    const float2 v = st[i];
    se += v.y * exp2_approx((v.x - mx) * k2);
    if (zsum != nullptr) zs += zsum[at * halves + i];
  }
  se = warp_sum(se);
  if (zsum != nullptr) zs = warp_sum(zs);
  if (lane != 0) return;
  const float log2_se = log2f(se), lse2 = fmaf(mx, k2, log2_se);
  c.lse2[row] = lse2;
  const int src = c.src[row];
  if (src < 0) return;
  // lse - z_y from the difference to the maximum: the size of the logits does not enter its error
  float loss = c.scale * (mx - zt[at]) + log2_se * kLn2;
  const float lse = lse2 * kLn2;
  if (c.smooth > 0.f) loss += c.smooth * (c.scale * zt[at] - zs / static_cast<float>(c.V));
  f.rows[src] = c.sign * (loss + c.z * lse * lse);
}

__global__ void __launch_bounds__(1024) vl_total_k(const VlCall c, const VlForward f) {
  __shared__ float part[32];
  grid_dependency_wait();
  float s = 0.f;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < c.T; i += 1024) s += f.rows[i];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_sum(part[threadIdx.x]);
    if (threadIdx.x == 0) *f.total = s * *c.ginv;
  }
}

// dh in the call's order: the K slices' sum of a counted row, 0 of the others.  The target's
// gradient, about -1 beside words' of some 1 / V, is most of a row's: what rounding it to bf16
// took (resid) is added back as resid w_target, so that its error is not dh's.
__global__ void __launch_bounds__(256) vl_scatter_k(const VlCall c, const float* acc, int ldc,
                                                    int64_t slice, int slices, const float* resid,
                                                    const float* alpha, __nv_bfloat16* dh) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, nv = c.H >> 3;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < c.T;
       row += static_cast<int64_t>(gridDim.x) * 8) {
    const int at = c.pos[row];
    uint4* out = reinterpret_cast<uint4*>(dh + row * c.H);
    const float r = at >= 0 ? resid[at] * *alpha : 0.f;
    const uint4* w =
        reinterpret_cast<const uint4*>(c.w + static_cast<int64_t>(at >= 0 ? c.target[at] : 0) * c.H);
#pragma unroll 2
    for (int i = lane; i < nv; i += 32) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (at >= 0) {
        const uint4 t = w[i];
        const float2 t0 = unpack_bf16x2(t.x), t1 = unpack_bf16x2(t.y), t2 = unpack_bf16x2(t.z),
                     t3 = unpack_bf16x2(t.w);
        float4 a = make_float4(r * t0.x, r * t0.y, r * t1.x, r * t1.y);
        float4 b = make_float4(r * t2.x, r * t2.y, r * t3.x, r * t3.y);
        const float* p = acc + static_cast<int64_t>(at) * ldc + i * 8;
        for (int k = 0; k < slices; ++k) {
          const float4 x = *reinterpret_cast<const float4*>(p + k * slice);
          const float4 y = *reinterpret_cast<const float4*>(p + k * slice + 4);
          a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
          b.x += y.x; b.y += y.y; b.z += y.z; b.w += y.w;
        }
        u = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y),
                       pack_bf16x2(b.z, b.w));
      }
      out[i] = u;
    }
  }
}

// What the rows' gradients of the logits leave out: scale, sign and unit, and the loss's own factor
// where the rows share it.
__global__ void vl_alpha_k(const VlCall c, const float* gout, bool per_row, float unit,
                           float* alpha) {
  grid_dependents_go();
  *alpha = c.scale * c.sign * unit * (per_row ? 1.f : *gout * *c.ginv);
}
float unit_of(const VlCall& c) { return c.smooth < 1.f ? 1.f - c.smooth : 1.f; }

int pad32(int n) { return (n + 31) / 32 * 32; }
int halves_of(const VlCall& c) { return 2 * ((c.V + 255) / 256); }

GemmEpi epi_of(const VlCall& c) {
  GemmEpi ep;
  ep.ce.k2 = c.scale * kLog2e;
  ep.ce.scale = c.scale;
  ep.ce.target = c.target;
  ep.ce.n_valid = 0;
  ep.m_dev = c.cnt + 1;
  ep.dependent = 1;
  return ep;
}

}  // namespace

// Rows whose statistics are held at a time: about 256 MB of them, whole row tiles.
static int64_t rows_each(const VlCall& c) {
  const int64_t R = vl_rows(c.T), row = static_cast<int64_t>(halves_of(c)) * 12;
  const int64_t n = std::max<int64_t>(1, (256 << 20) / row / 256) * 256;
  return std::min(R, n);
}

int64_t vl_forward_floats(const VlCall& c) {
  return rows_each(c) * (static_cast<int64_t>(halves_of(c)) * (c.smooth > 0.f ? 3 : 2) + 1);
}

int vl_forward(const VlCall& c, const VlForward& f, cudaStream_t s) {
  const int64_t R = vl_rows(c.T), each = rows_each(c);
  const int halves = halves_of(c);
  // rows a block: enough blocks to copy with every SM, few enough that the counting stays small
  int per = static_cast<int>((c.T + 2 * c.num_sms - 1) / (2 * c.num_sms));
  per = per < 8 ? 8 : per > 256 ? 256 : per;
  const int64_t most = static_cast<int64_t>(4) * c.num_sms, turns = (c.T + 255) / 256;
  if (turns > most) per = static_cast<int>((turns + most - 1) / most) * 256;
  vl_gather_k<<<static_cast<unsigned>((c.T + per - 1) / per), 256, 0, s>>>(c, f, per);
  float2* stats = reinterpret_cast<float2*>(f.ws);
  float* zsum = c.smooth > 0.f ? f.ws + 2 * each * halves : nullptr;
  float* zt = f.ws + each * halves * (c.smooth > 0.f ? 3 : 2);
  for (int64_t r0 = 0; r0 < R; r0 += each) {
    const int64_t n = std::min(each, R - r0);
    GemmArgs g;
    g.A = c.hc + r0 * c.H;
    g.lda = c.H;
    g.B = c.w;
    g.ldb = c.H;
    g.M = static_cast<int>(n);
    g.N = pad32(c.V);
    g.n_valid = c.V;
    g.K = c.H;
    g.epi = EPI_CE_FWD;
    g.bn = 256;
    g.num_sms = c.num_sms;
    GemmEpi ep = epi_of(c);
    ep.m_off = static_cast<int>(r0);
    ep.ce.target = c.target + r0;
    ep.ce.stats = stats;
    ep.ce.zt = zt;
    ep.ce.zsum = zsum;
    ep.ce.n_valid = c.V;
    ep.group_m = 8;
    int rc = gemm_tc_launch(g, ep, s, c.err);
    if (rc) return rc;
    rc = launch_dependent(vl_rows_k, dim3(static_cast<unsigned>((n + 7) / 8)), 256, s, c, f, stats,
                          zt, zsum, halves, r0, n);
    if (rc) return rc;
  }
  if (f.total != nullptr) {
    const int rc = launch_dependent(vl_total_k, dim3(1), 1024, s, c, f);
    if (rc) return rc;
  }
  return static_cast<int>(cudaGetLastError());
}

// The pieces of the vocabulary and the K slices of the hidden gradient.
//
// One piece where the workspace holds all of dz; else about 256 MB of it, but at least 4096 words:
// of two L2 caches' worth the next product still finds some, while every piece costs three launches
// and dh read and written once more.  Back to back at the power limit, 32768 x 32000 x 896 in 128,
// 256, 512, 2048 MB of workspace: 8.8, 6.9, 6.9, 6.5 ms (the last is one piece, in four times the
// memory); 4096 x 100000 x 4096 in 64, 192, 256, 512 MB: 10.5, 10.2, 10.1, 10.1 ms; one piece against
// two of 3001 x 50021 x 1024: 0.93, 1.01 ms.  With more rows the pieces get smaller: 131072 rows of
// 32000 x 896 take 16 of them, 34.7 ms, of which the 470 MB of dh that each reads and writes are 2.
//
// dh has few tiles (256 x 256, one CTA pair each): 48 at 3000 x 1024 for 74 pairs.  It is cut along
// the words into the slices that fill the waves of pairs best; as the counted rows may be any part
// of all, the rule takes the mean over all, three quarters and half of them.
void vl_backward_plan(const VlCall& c, int64_t workspace_bytes, VlBackward* b) {
  const int64_t R = vl_rows(c.T);
  int64_t words = std::max<int64_t>(workspace_bytes / (2 * R) / 256 * 256, 256);
  if (words < c.V) words = std::min(words, std::max<int64_t>((128 << 20) / R / 256 * 256, 4096));
  const int64_t pieces = (c.V + words - 1) / words;
  b->piece = static_cast<int>(((c.V + pieces - 1) / pieces + 255) / 256 * 256);
  const double rate = 1.4e9, hbm = 6.5e6;  // operations and bytes a us
  const int64_t cols = (c.H + 255) / 256;
  const int64_t units = R > 128 ? c.num_sms / 2 : c.num_sms;
  // slices of at least eight K blocks, and some of the last piece's for each
  words = std::min<int64_t>(b->piece, c.V);
  const int64_t last = (c.V - (c.V - 1) / b->piece * b->piece + 63) / 64;
  const int64_t top = std::min<int64_t>(std::min<int64_t>(words / 512, last), 64);
  double best = 0;
  b->ksplit = 1;
  for (int64_t ks = 1; ks <= std::max<int64_t>(1, top); ++ks) {
    double us = 0;
    for (int part = 2; part <= 4; ++part) {
      const int64_t rows = std::max<int64_t>(1, R * part / 4);
      const int64_t tiles = (R > 128 ? (rows + 255) / 256 : 1) * cols * ks;
      const double tile = 2.0 * (R > 128 ? 256 : 128) * 256 * static_cast<double>(words) / ks;
      us += static_cast<double>((tiles + units - 1) / units * units) * tile / rate +
            static_cast<double>(ks) * rows * pad32(c.H) * 8 / hbm;
    }
    if (best == 0 || us < 0.97 * best) {
      best = us;
      b->ksplit = static_cast<int>(ks);
    }
  }
}

int64_t vl_acc_floats(const VlCall& c, const VlBackward& b) {
  return static_cast<int64_t>(b.ksplit) * vl_rows(c.T) * pad32(c.H);
}

int vl_backward(const VlCall& c, const VlBackward& b, cudaStream_t s) {
  const int64_t R = vl_rows(c.T);
  const int ldh = pad32(c.H);
  vl_alpha_k<<<1, 1, 0, s>>>(c, b.gout, b.per_row, unit_of(c), b.alpha);
  for (int v0 = 0; v0 < c.V; v0 += b.piece) {
    const int n = c.V - v0 < b.piece ? c.V - v0 : b.piece;
    const __nv_bfloat16* w = c.w + static_cast<int64_t>(v0) * c.H;
    GemmArgs g;
    g.num_sms = c.num_sms;
    // dz of the piece
    g.A = c.hc;
    g.lda = c.H;
    g.B = w;
    g.ldb = c.H;
    g.M = static_cast<int>(R);
    g.N = pad32(n);
    g.n_valid = n;
    g.K = c.H;
    g.epi = EPI_CE_GRAD;
    g.bn = 256;
    GemmEpi ep = epi_of(c);
    ep.c = b.dl;
    ep.ldc = b.piece;
    ep.ce.lse2 = c.lse2;
    ep.ce.gout = b.per_row ? b.gout : nullptr;
    ep.ce.inv_unit = 1.f / unit_of(c);
    ep.ce.src = c.src;
    ep.ce.z2 = 2.f * c.z;
    ep.ce.smooth = c.smooth;
    ep.ce.smooth_v = c.smooth / static_cast<float>(c.V);
    ep.ce.col0 = v0;
    ep.ce.resid = b.resid;
    ep.ce.n_valid = n;
    ep.group_m = 8;
    int rc = gemm_tc_launch(g, ep, s, c.err);
    if (rc) return rc;
    if (b.dh != nullptr) {  // dh (+)= dz W
      GemmArgs d;
      d.num_sms = c.num_sms;
      d.A = b.dl;
      d.lda = b.piece;
      d.B = w;
      d.ldb = c.H;
      d.b_mn = true;
      d.M = static_cast<int>(R);
      d.N = ldh;
      d.n_valid = c.H;
      d.K = n;
      d.ksplit = b.ksplit;
      d.epi = v0 == 0 ? EPI_F32 : EPI_F32_ACC;
      GemmEpi e;
      e.m_dev = c.cnt + 1;
      e.c = b.acc;
      e.ldc = ldh;
      e.split_stride = R * ldh;
      e.alpha_dev = b.alpha;
      e.dependent = 1;
      rc = gemm_tc_launch(d, e, s, c.err);
      if (rc) return rc;
    }
    if (b.dw != nullptr) {  // dW of the piece = dz^T h
      GemmArgs d;
      d.num_sms = c.num_sms;
      d.A = b.dl;
      d.lda = b.piece;
      d.a_mn = true;
      d.B = c.hc;
      d.ldb = c.H;
      d.b_mn = true;
      d.M = n;
      d.N = ldh;
      d.n_valid = c.H;
      d.K = static_cast<int>(R);
      d.epi = EPI_STORE;
      GemmEpi e;
      e.k_dev = c.cnt + 1;
      e.alpha_dev = b.alpha;
      e.dependent = 1;
      e.c = b.dw + static_cast<int64_t>(v0) * c.H;
      e.ldc = c.H;
      rc = gemm_tc_launch(d, e, s, c.err);
      if (rc) return rc;
    }
  }
  if (b.dh != nullptr) {
    const int64_t want = (c.T + 7) / 8, most = static_cast<int64_t>(c.num_sms) * 8;
    const int rc =
        launch_dependent(vl_scatter_k, dim3(static_cast<unsigned>(want < most ? want : most)), 256, s,
                         c, b.acc, ldh, R * ldh, b.ksplit, b.resid, b.alpha, b.dh);
    if (rc) return rc;
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace cfb
