// The 8-bit paged KV cache: quantising append, read-back, eviction (sm_100a).
//
// A block is one page (16 tokens) of one head's keys or values, with one fp32 scale s;
// a code c stands for c * s.  All these kernels move bytes: what bounds them is HBM
// bandwidth for long inputs and launch latency for a decode step.
// Measured (8 heads, D 128): append of 4 x 2048 tokens 13.5 us and its read-back 11.8 us (each
// profiled alone), 20.4 us as two calls; a read-back of 3.1 GB 480 us (6.5 TB/s); a move of
// 2.06 GB 365 us (5.6 TB/s); selection in 2048 rows of 1500 to 4096 masses 45 us; append of 64 tokens 2.8 us.
#include "paged8.cuh"

namespace cfb {
namespace {

constexpr unsigned kFull = 0xffffffffu;

// ---------------------------------------------------------------------------- append
// For the new tokens x of a block with scale s0 (0 when it holds no older token):
//   s = max(s0, max|x| / levels), code = round(x / s), and where s > s0 the older codes
//   become round(code * s0 / s).
// One warp owns a (block, head, K or V): the block's maximum is one warp reduction and
// nothing is shared between warps.  A lane holds 8 values (16 bytes) of each of D / 16
// loads, all issued before the reduction.  max|x| is taken on the 16-bit patterns, which
// order as the magnitudes do and let a NaN through to the scale.  Long chunks are bound by
// instructions as much as by bytes, hence the packed maxima.
//
// Blocks are enumerated without reading lengths on the host: sequence i either has a row of
// the grid, as long as the blocks a chunk of max_q_len can touch, or, when chunks are uneven,
// the items from floor(cu_q[i] / 16) + 2 i on, which leaves room for its at most
// floor(q / 16) + 2 blocks; the host takes the smaller enumeration.
// A block with a value that is not finite has a scale that is not, and codes of 0.
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(256, 3)
    p8_append_kernel(P8Cache c, P8Seqs s, const T* __restrict__ k, int64_t k_stride,
                     const T* __restrict__ v, int64_t v_stride, int64_t N, unsigned units,
                     int per_seq, int max_q_len, float* __restrict__ mass, int* err) {
  constexpr int CH = D / 8;        // lanes of a row
  constexpr int RPL = 32 / CH;     // rows of one load
  constexpr int NL = kP8Page / RPL;
  const unsigned unit = blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  p8_grid_wait();
  if (unit >= units) return;
  const int hx = static_cast<int>(unit % (2 * c.Hkv));
  int64_t j = unit / (2 * c.Hkv);
  int seq = blockIdx.y;
  if (per_seq == 0) {
    int lo = 0, hi = s.num_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(s.cu_q + mid) / kP8Page + 2 * static_cast<int64_t>(mid) <= j) lo = mid;
      else hi = mid - 1;
    }
    seq = lo;
    j -= __ldg(s.cu_q + seq) / kP8Page + 2 * static_cast<int64_t>(seq);
    if (j < 0) return;  // rows before cu_q[0] are not this call's
  }
  const int row0 = __ldg(s.cu_q + seq);
  const int q_len = __ldg(s.cu_q + seq + 1) - row0;
  const int kv = p8_len(s.kv_lens, seq, s.max_pages, err, 60);
  const int start = kv - q_len;                       // position of row0's token
  const int first = max(start, 0);
  const int64_t blk = first / kP8Page + j;
  if (q_len <= 0 || blk * kP8Page >= kv) return;
  if (q_len > max_q_len && lane == 0) report_error(err, kErrBounds, 59);
  if (row0 < 0 || static_cast<int64_t>(row0) + q_len > N) {
    if (lane == 0) report_error(err, kErrBounds, 61);
    return;
  }
  const int base = static_cast<int>(blk) * kP8Page;
  const int lo = max(first, base) - base, hi = min(kv - base, kP8Page);  // new tokens of the block
  const int h = hx >> 1, x = hx & 1;
  const T* src = x ? v : k;
  const int64_t stride = x ? v_stride : k_stride;
  const int r = lane / CH, col = (lane % CH) * 8;

  uint4 in[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int t = i * RPL + r;
    in[i] = make_uint4(0, 0, 0, 0);
    if (t >= lo && t < hi)
      in[i] = __ldg(reinterpret_cast<const uint4*>(
          src + static_cast<int64_t>(row0 + base + t - start) * stride + h * D + col));
  }
  // after the loads: its check waits for the table
  const int64_t page = p8_page(s.table + static_cast<int64_t>(seq) * s.max_pages,
                               static_cast<int>(blk), c.num_pages, err, 62);
  const int64_t ph = (page * c.Hkv + h) * 2 + x;
  float* scale = c.scales + ph;
  uint8_t* codes = c.codes + ph * (kP8Page * D);
  const float s0 = lo > 0 ? *scale : 0.f;
  // magnitudes as pairs of 16-bit patterns: three instructions for four values
  uint32_t top2 = 0;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    top2 = __vimax3_u16x2(top2, in[i].x & 0x7fff7fffu, in[i].y & 0x7fff7fffu);
    top2 = __vimax3_u16x2(top2, in[i].z & 0x7fff7fffu, in[i].w & 0x7fff7fffu);
  }
  const uint32_t top = __reduce_max_sync(kFull, max(top2 & 0xffffu, top2 >> 16));
  const float sn = __fdiv_rn(P8Io<T>::unpack(top).x, p8_levels<FMT>());
  const float sc = (sn > s0 || sn != sn) ? sn : s0;
  const bool fine = sc <= 3.402823466e38f;
  const float inv = fine && sc > 0.f ? __fdiv_rn(1.f, sc) : 0.f;
  auto store = [&](auto scaled) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int t = i * RPL + r;
      if (t < lo || t >= hi) continue;
      const uint32_t w[4] = {in[i].x, in[i].y, in[i].z, in[i].w};
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 q = scaled(P8Io<T>::unpack(w[e]));
        f[2 * e] = q.x;
        f[2 * e + 1] = q.y;
      }
      *reinterpret_cast<uint2*>(codes + t * D + col) =
          make_uint2(p8_from_float<FMT>(f), p8_from_float<FMT>(f + 4));
    }
  };
  if (!fine)
    store([](float2) { return make_float2(0.f, 0.f); });
  else if (isinf(inv))  // a subnormal scale
    store([&](float2 x) { return make_float2(__fdiv_rn(x.x, sc), __fdiv_rn(x.y, sc)); });
  else
    // scalar products: a packed one would be fused with the adder's rounding, and codes would
    // differ from the formula's at ties
    store([&](float2 x) { return make_float2(__fmul_rn(x.x, inv), __fmul_rn(x.y, inv)); });
  if (lo > 0 && sc != s0) {  // the scale grew: the older codes follow it
    const float ratio = fine && sc > 0.f ? __fdiv_rn(s0, sc) : 0.f;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int t = i * RPL + r;
      if (t >= lo) continue;
      uint2* at = reinterpret_cast<uint2*>(codes + t * D + col);
      const uint2 old = *at;
      float f[8];
      p8_to_float<FMT>(old.x, f);
      p8_to_float<FMT>(old.y, f + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __fmul_rn(f[e], ratio);
      *at = make_uint2(p8_from_float<FMT>(f), p8_from_float<FMT>(f + 4));
    }
  }
  if (lane == 0 && (sc != s0 || lo == 0)) *scale = sc;
  if (mass != nullptr && x == 0 && lane >= lo && lane < hi)
    mass[(page * c.Hkv + h) * kP8Page + lane] = 0.f;
}

// ------------------------------------------------------------------------------ read
// One warp per (layer, sequence, page, head, K or V): 8 codes a lane and load, so that its
// 16-byte stores are dense; the values are rounded once to the output's type.
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(256)
    p8_read_kernel(P8Cache c, P8Seqs s, unsigned units, T* __restrict__ k_out,
                   T* __restrict__ v_out, int* err) {
  constexpr int NC = kP8Page * D / 8 / 32;  // 8-code pieces of a lane
  const unsigned unit = blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int x = unit & 1, h = (unit >> 1) % c.Hkv, blk = (unit >> 1) / c.Hkv;
  const int seq = blockIdx.y;
  const int64_t layer = blockIdx.z;
  p8_grid_wait();
  if (unit >= units) return;
  // the table's entry beside the length that says whether it counts
  const int entry = __ldg(s.table + static_cast<int64_t>(seq) * s.max_pages + blk);
  const int kv = p8_len(s.kv_lens, seq, s.max_pages, err, 63);
  const int live = min(kv - blk * kP8Page, kP8Page);  // tokens of the block, may be <= 0
  const int64_t Lp = static_cast<int64_t>(s.max_pages) * kP8Page;
  T* dst = (x ? v_out : k_out) +
           (((layer * s.num_seqs + seq) * c.Hkv + h) * Lp + blk * kP8Page) * D;
  const uint8_t* src = nullptr;
  float sc = 0.f;
  if (live > 0) {
    const int64_t page = p8_checked(entry, c.num_pages, err, 64);
    const int64_t ph = ((layer * c.num_pages + page) * c.Hkv + h) * 2 + x;
    sc = __ldg(c.scales + ph);
    src = c.codes + ph * (kP8Page * D);
  }
  uint2 w[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int e = (i * 32 + lane) * 8;
    w[i] = e / D < live ? __ldg(reinterpret_cast<const uint2*>(src + e)) : make_uint2(0, 0);
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int e = (i * 32 + lane) * 8;
    uint4 a = make_uint4(0, 0, 0, 0);
    if (e / D < live) {
      float f[8];
      p8_to_float<FMT>(w[i].x, f);
      p8_to_float<FMT>(w[i].y, f + 4);
      a = make_uint4(P8Io<T>::pack(f[0] * sc, f[1] * sc), P8Io<T>::pack(f[2] * sc, f[3] * sc),
                     P8Io<T>::pack(f[4] * sc, f[5] * sc), P8Io<T>::pack(f[6] * sc, f[7] * sc));
    }
    *reinterpret_cast<uint4*>(dst + e) = a;
  }
}

// ----------------------------------------------------------------------------- evict
// Select: one CTA per (layer, sequence, head) finds the k = budget - recent largest of
// the n = len - recent older masses by a radix select on order-preserving 32-bit keys
// (digits of 11, 11 and 10 bits, each a histogram in shared memory; it ends early once a
// digit's keys are all kept), then writes the kept indices in order: everything above the
// k-th key, and of its equals the lowest indices.  The first digit covers the exponent and
// two bits more: masses crowd into few exponents, and the histogram's atomics would queue.
constexpr int kSelThreads = 256;
constexpr int kSelBins = 2048;
constexpr int kSelKeys = 40 * 1024;  // keys held in shared memory; longer rows re-read global

__device__ __forceinline__ uint32_t mass_key(float m) {
  const uint32_t u = __float_as_uint(m + 0.f);  // -0 and 0 are one key
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Exclusive sums over the CTA's threads of two counts, in thread order.
__device__ __forceinline__ int2 sums_before(int2 v, int2 (&s_part)[kSelThreads / 32]) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int2 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(kFull, inc.x, o), b = __shfl_up_sync(kFull, inc.y, o);
    if (lane >= o) {
      inc.x += a;
      inc.y += b;
    }
  }
  if (lane == 31) s_part[warp] = inc;
  __syncthreads();
  int2 r = make_int2(inc.x - v.x, inc.y - v.y);
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w)
    if (w < warp) {
      r.x += s_part[w].x;
      r.y += s_part[w].y;
    }
  return r;
}

__global__ void __launch_bounds__(kSelThreads)
    p8_select_kernel(P8Cache c, P8Seqs s, const float* __restrict__ mass, int budget, int recent,
                     int32_t* __restrict__ keep, int cap, int* err) {
  extern __shared__ uint32_t s_keys[];
  __shared__ int s_hist[kSelBins];
  __shared__ int2 s_part[2][kSelThreads / 32];
  __shared__ int s_digit, s_need, s_count;
  const int h = blockIdx.x, seq = blockIdx.y;
  const int64_t layer = blockIdx.z;
  const int tid = threadIdx.x;
  p8_grid_wait();
  const int len = p8_len(s.kv_lens, seq, s.max_pages, err, 65);
  int32_t* row = keep + ((layer * s.num_seqs + seq) * c.Hkv + h) * budget;
  if (len <= budget) {
    for (int i = tid; i < budget; i += kSelThreads) row[i] = i < len ? i : -1;
    return;
  }
  const int n = len - recent, k = budget - recent;
  for (int i = tid; i < recent; i += kSelThreads) row[k + i] = n + i;
  if (k == 0) return;
  const int32_t* table = s.table + static_cast<int64_t>(seq) * s.max_pages;
  const float* m = mass + layer * c.num_pages * c.Hkv * kP8Page;
  auto fetch = [&](int i) {
    const int64_t page = p8_page(table, i / kP8Page, c.num_pages, err, 66);
    return mass_key(__ldg(m + (page * c.Hkv + h) * kP8Page + i % kP8Page));
  };
  const bool held = n <= cap;
  if (held) {
#pragma unroll 4
    for (int i = tid; i < n; i += kSelThreads) s_keys[i] = fetch(i);
  }
  auto key = [&](int i) { return held ? s_keys[i] : fetch(i); };
  uint32_t prefix = 0, mask = 0;
  int need = k;  // of the keys that match the prefix, how many are kept
  int shift = 32;
#pragma unroll
  for (int digit = 0; digit < 3; ++digit) {
    const int bits = digit < 2 ? 11 : 10, bins = 1 << bits;
    shift -= bits;
    for (int i = tid; i < bins; i += kSelThreads) s_hist[i] = 0;
    __syncthreads();  // also: the keys are there
    for (int i = tid; i < n; i += kSelThreads) {
      const uint32_t u = key(i);
      if ((u & mask) == prefix) atomicAdd(&s_hist[(u >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    // the digit at which the count from the top first reaches `need`
    const int each = bins / kSelThreads;
    int cnt[8], sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      cnt[i] = i < each ? s_hist[bins - 1 - (tid * each + i)] : 0;
      sum += cnt[i];
    }
    int before = sums_before(make_int2(sum, 0), s_part[digit & 1]).x;
    if (before < need && before + sum >= need) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (before < need && before + cnt[i] >= need) {
          s_digit = bins - 1 - (tid * each + i);
          s_need = need - before;
          s_count = cnt[i];
          before = need;  // found
        } else {
          before += cnt[i];
        }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(s_digit) << shift;
    mask |= static_cast<uint32_t>(bins - 1) << shift;
    need = s_need;
    if (s_count == need) break;  // all that match are kept
  }
  // ordered write: each thread owns a contiguous stretch of the older tokens
  const int per = (n + kSelThreads - 1) / kSelThreads;
  const int a = min(n, tid * per), b = min(n, a + per);
  int gt = 0, eq = 0;
  for (int i = a; i < b; ++i) {
    const uint32_t u = key(i) & mask;
    gt += u > prefix;
    eq += u == prefix;
  }
  __syncthreads();  // the partial sums of the last digit are read
  const int2 at = sums_before(make_int2(gt, eq), s_part[0]);
  gt = at.x;
  eq = at.y;
  for (int i = a; i < b; ++i) {
    const uint32_t u = key(i) & mask;
    if (u > prefix || (u == prefix && eq < need)) row[gt + min(eq, need)] = i;
    gt += u > prefix;
    eq += u == prefix;
  }
}

// Move: one warp per (layer, sequence, head, new block).  The block's scale is the
// largest among its tokens' old blocks, so a token from that block keeps its codes and
// the others are rounded once more: code = round(code * s_old / s).
template <int FMT, int D>
__global__ void __launch_bounds__(256)
    p8_move_kernel(P8Cache c, P8Seqs s, float* __restrict__ mass, int layers,
                   const int32_t* __restrict__ dst_table, int dst_pages, int budget,
                   const int32_t* __restrict__ keep, unsigned units, int* err) {
  constexpr int CPR = D / 16;                 // 16-code chunks of a row
  constexpr int NC = 2 * kP8Page * CPR / 32;  // chunks of a lane, K and V
  const unsigned unit = blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int h = unit % c.Hkv, blk = unit / c.Hkv, seq = blockIdx.y;
  const int64_t layer = blockIdx.z;
  p8_grid_wait();
  if (unit >= units) return;
  const int len = p8_len(s.kv_lens, seq, s.max_pages, err, 67);
  const int kept = min(len, budget);
  const int live = min(kept - blk * kP8Page, kP8Page);
  if (live <= 0) return;
  if (blk == dst_pages - 1 && kept > dst_pages * kP8Page && lane == 0)
    report_error(err, kErrBounds, 58);  // the new pages are too few
  const int64_t dpage = p8_page(dst_table + static_cast<int64_t>(seq) * dst_pages, blk,
                                c.num_pages, err, 68);
  const int64_t dph = (layer * c.num_pages + dpage) * c.Hkv + h;
  const int32_t* row = keep + ((layer * s.num_seqs + seq) * c.Hkv + h) * budget + blk * kP8Page;
  // lanes 0-15 look up the block's tokens
  int64_t sph = 0;
  int off = 0;
  float2 sc = make_float2(0.f, 0.f);
  float m = 0.f;
  if (lane < live) {
    const int i = __ldg(row + lane);
    const int64_t page = p8_page(s.table + static_cast<int64_t>(seq) * s.max_pages, i / kP8Page,
                                 c.num_pages, err, 69);
    sph = (layer * c.num_pages + page) * c.Hkv + h;
    off = i % kP8Page;
    sc = __ldg(reinterpret_cast<const float2*>(c.scales) + sph);
    if (mass != nullptr) m = mass[sph * kP8Page + off];
  }
  uint32_t kb = __float_as_uint(sc.x), vb = __float_as_uint(sc.y);  // scales are >= 0 or NaN
  kb = __reduce_max_sync(kFull, kb);
  vb = __reduce_max_sync(kFull, vb);
  const float top[2] = {__uint_as_float(kb), __uint_as_float(vb)};
  uint4 w[NC];
  float ratio[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int e = i * 32 + lane;
    const int x = e / (kP8Page * CPR), t = e / CPR % kP8Page, ch = e % CPR;
    const int64_t p = __shfl_sync(kFull, sph, t);
    const int o = __shfl_sync(kFull, off, t);
    const float so = x ? __shfl_sync(kFull, sc.y, t) : __shfl_sync(kFull, sc.x, t);
    w[i] = make_uint4(0, 0, 0, 0);
    if (t < live)
      w[i] = __ldg(reinterpret_cast<const uint4*>(c.codes + ((p * 2 + x) * kP8Page + o) * D) + ch);
    ratio[i] = so == top[x] ? 1.f : __fdiv_rn(so, top[x]);
    if (ratio[i] != ratio[i]) ratio[i] = 0.f;  // a scale that is not a number: codes of 0
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    if (ratio[i] != 1.f) {
      uint32_t* q = reinterpret_cast<uint32_t*>(&w[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[4];
        p8_to_float<FMT>(q[j], f);
#pragma unroll
        for (int z = 0; z < 4; ++z) f[z] = __fmul_rn(f[z], ratio[i]);
        q[j] = p8_from_float<FMT>(f);
      }
    }
    reinterpret_cast<uint4*>(c.codes + dph * (2 * kP8Page * D))[i * 32 + lane] = w[i];
  }
  if (lane == 0) reinterpret_cast<float2*>(c.scales)[dph] = make_float2(top[0], top[1]);
  if (mass != nullptr && lane < kP8Page) mass[dph * kP8Page + lane] = m;
}

template <typename T, int FMT, int D>
int launch_append(const P8Cache& c, const P8Seqs& s, const void* k, int64_t ks, const void* v,
                  int64_t vs, int64_t N, unsigned units, int per_seq, int max_q_len, float* mass,
                  int* err, cudaStream_t st) {
  return p8_launch(p8_append_kernel<T, FMT, D>,
                   dim3((units + 7) / 8, per_seq > 0 ? s.num_seqs : 1), 256, 0, st, c, s,
                   static_cast<const T*>(k), ks, static_cast<const T*>(v), vs, N, units, per_seq,
                   max_q_len, mass, err);
}

}  // namespace

#define CFB_P8_TYPES(CALL)                                     \
  do {                                                         \
    const int key_ = type * 4 + c.fmt * 2 + (c.D == 128);      \
    switch (key_) {                                            \
      case 0: CALL(__nv_bfloat16, kP8Int8, 64); break;         \
      case 1: CALL(__nv_bfloat16, kP8Int8, 128); break;        \
      case 2: CALL(__nv_bfloat16, kP8E4m3, 64); break;         \
      case 3: CALL(__nv_bfloat16, kP8E4m3, 128); break;        \
      case 4: CALL(__half, kP8Int8, 64); break;                \
      case 5: CALL(__half, kP8Int8, 128); break;               \
      case 6: CALL(__half, kP8E4m3, 64); break;                \
      case 7: CALL(__half, kP8E4m3, 128); break;               \
      default: return -2;                                      \
    }                                                          \
  } while (0)

int p8_append(const P8Cache& c, const P8Seqs& s, const void* k, int64_t k_stride, const void* v,
              int64_t v_stride, int64_t N, int max_q_len, int type, float* mass, int* err,
              cudaStream_t stream) {
  if (N <= 0 || s.num_seqs <= 0) return 0;
  const int64_t per_seq = (max_q_len + kP8Page - 2) / kP8Page + 1;
  const int64_t even = per_seq * s.num_seqs, uneven = N / kP8Page + 2 * s.num_seqs;
  const int64_t items = even <= uneven ? even : uneven;
  const int ps = even <= uneven ? static_cast<int>(per_seq) : 0;
  const int64_t units = (ps ? per_seq : items) * 2 * c.Hkv;
  if (units > 0x7fffffff) return -3;
  int rc = 0;
#define CFB_CALL(T, F, DD)                                                                       \
  rc = launch_append<T, F, DD>(c, s, k, k_stride, v, v_stride, N, static_cast<unsigned>(units), ps, \
                               max_q_len, mass, err, stream)
  CFB_P8_TYPES(CFB_CALL);
#undef CFB_CALL
  return rc ? rc : static_cast<int>(cudaGetLastError());
}

int p8_read(const P8Cache& c, const P8Seqs& s, int layers, void* k_out, void* v_out, int type,
            int* err, cudaStream_t stream) {
  const int64_t units = static_cast<int64_t>(s.max_pages) * c.Hkv * 2;
  if (layers <= 0 || s.num_seqs <= 0) return 0;
  if (units > 0x7fffffff) return -3;
  const dim3 grid(static_cast<unsigned>((units + 7) / 8), s.num_seqs, layers);
  int rc = 0;
#define CFB_CALL(T, F, DD)                                                              \
  rc = p8_launch(p8_read_kernel<T, F, DD>, grid, 256, 0, stream, c, s,                   \
                 static_cast<unsigned>(units), static_cast<T*>(k_out), static_cast<T*>(v_out), err)
  CFB_P8_TYPES(CFB_CALL);
#undef CFB_CALL
  return rc ? rc : static_cast<int>(cudaGetLastError());
}

int p8_evict(const P8Cache& c, const P8Seqs& s, float* mass, int layers, const int32_t* dst_table,
             int dst_pages, int budget, int recent, int32_t* keep, int* err,
             cudaStream_t stream) {
  if (s.num_seqs <= 0 || layers <= 0) return 0;
  if (s.num_seqs > 65535 || layers > 65535) return -3;
  const int64_t units = static_cast<int64_t>(dst_pages) * c.Hkv;
  if (units > 0x7fffffff) return -3;
  const int longest = s.max_pages * kP8Page;
  const int cap = longest < kSelKeys ? longest : kSelKeys;
  const int smem = cap * 4;
  int rc = p8_opt_in<p8_select_kernel>(kSelKeys * 4);
  if (!rc)
    rc = p8_launch(p8_select_kernel, dim3(c.Hkv, s.num_seqs, layers), kSelThreads, smem, stream, c,
                   s, mass, budget, recent, keep, cap, err);
  if (rc) return rc;
  const dim3 grid(static_cast<unsigned>((units + 7) / 8), s.num_seqs, layers);
  const int type = kP8Bf16;
#define CFB_CALL(T, F, DD)                                                                  \
  rc = p8_launch(p8_move_kernel<F, DD>, grid, 256, 0, stream, c, s, mass, layers, dst_table, \
                 dst_pages, budget, keep, static_cast<unsigned>(units), err)
  CFB_P8_TYPES(CFB_CALL);
#undef CFB_CALL
  return rc ? rc : static_cast<int>(cudaGetLastError());
}

}  // namespace cfb
