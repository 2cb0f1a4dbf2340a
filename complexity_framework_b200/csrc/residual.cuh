// The joins of the residual stream: a branch's norm, its gate and residual scale, dropout, the
// sum and the next block's norm in one pass each way; and dropout by itself.
//
//   n = w1 * b / rms(b)      (n = b without w1)
//   x' = x + scale * m * gate * n,     m = 0 (dropped) or 65536 / (65536 - threshold)
//   y = w2 * x' / rms(x')
//
// Gradients, with xh = x' / rms(x'), bh = b / rms(b) (bh = b without w1) and means over a row:
//
//   g = dx' + (w2 dy - xh mean(w2 dy xh)) / rms(x'),          dx = g,   dw2 = sum_rows dy xh
//   t = scale * m * g,   S = sum_rows t bh,                   dgate = w1 S,   dw1 = gate S
//   db = (t gate w1 - bh mean(t gate w1 bh)) / rms(b)         (t gate without w1)
//
// The forward reads x, b and writes x', y; the backward reads dx', dy, x', b and writes dx, db; the
// dropout mask is drawn again from its counter instead of being stored.  Memory would bound both;
// what bounds the backward is latency at low occupancy, as every element passes two sums in
// sequence: 126 registers leave an SM 16 warps, whose stalls are fixed latencies, shared memory and
// barriers, and of the 310 warp instructions for 32 blocks of eight elements (120 more for their
// dropout) a scheduler issues one every other cycle.  So a row's fixed work is spread over as many
// elements as registers allow, rows come through a ring of bulk copies, arithmetic is in pairs,
// and what a call leaves out is asked for outside the rows.  Sums run in fp32; results are rounded
// once, at their stores.  The backward takes xh from the stored x', rounded to the stream's type,
// and 1 / rms from before that rounding: in 16 bits its gradients are off by 0.0021 to 0.0025 (root
// mean square) where one rounding gives 0.0017; x' kept in 32 bits would be 2 bytes an element more
// to write and to read.
// The columns' sums stay in registers over all rows of a CTA, and one small kernel adds the CTAs'
// sums in a fixed order, so that equal calls give equal bits.
//
// us (TB/s), bf16, with norms and gate, on one B200 (a copy runs at 6.55 TB/s):
//   32768 x 896   forward 38 (6.2), with dropout 49 (4.8); backward 74 (4.8), 92 (3.8)
//   8191 x 4096   forward 47 (5.7), with dropout 53 (5.1); backward 81 (5.0), 85 (4.7)
//   20000 x 903   forward 40 (3.6), with dropout 53 (2.8); backward 81 (2.7), 93 (2.3)
//   dropout alone of 32768 x 896: 21 (5.5)
//
// Templates of one element type each; residual_bf16.cu, residual_half.cu and residual_float.cu
// instantiate them, residual.cu dispatches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "philox.cuh"
#include "residual.h"

namespace cfb {
namespace {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half(v); }
template <>
__device__ __forceinline__ float from_f(float v) { return v; }

constexpr int kMaxStages = 4;
constexpr int kMaxSmem = 226 * 1024;  // dynamic; the static part takes less than the last KB

// Eight elements, a block of the dropout generator, in 16-byte accesses.
template <typename T>
struct Oct {
  uint4 raw[sizeof(T) / 2];
  __device__ __forceinline__ void load_once(const T* p) {
#pragma unroll
    for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q)
      asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(raw[q].x), "=r"(raw[q].y), "=r"(raw[q].z), "=r"(raw[q].w)
                   : "l"(reinterpret_cast<const uint4*>(p) + q));
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q)
      raw[q] = __ldg(reinterpret_cast<const uint4*>(p) + q);
  }
  __device__ __forceinline__ void get(float2* v) const {
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = make_float2(to_f<T>(e[2 * j]), to_f<T>(e[2 * j + 1]));
  }
  static __device__ __forceinline__ void store(T* p, const float2* v) {
    uint4 u[sizeof(T) / 2];
    T* e = reinterpret_cast<T*>(u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      e[2 * j] = from_f<T>(v[j].x);
      e[2 * j + 1] = from_f<T>(v[j].y);
    }
#pragma unroll
    for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q)
      reinterpret_cast<uint4*>(p)[q] = u[q];
  }
};
template <>
__device__ __forceinline__ void Oct<__nv_bfloat16>::get(float2* v) const {
  const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
}
template <>
__device__ __forceinline__ void Oct<__nv_bfloat16>::store(__nv_bfloat16* p, const float2* v) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[1].x, v[1].y),
                 pack_bf16x2(v[2].x, v[2].y), pack_bf16x2(v[3].x, v[3].y));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

// Sum over the RT threads of a row.  `red` holds RT / 32 floats of this row's group; a row's two
// sums have their own, so that one barrier a sum is enough (see Feed::end).
template <int RT>
__device__ __forceinline__ float row_sum(float v, float* red, int group, int tid) {
  v = warp_sum(v);
  if constexpr (RT > 32) {
    if ((tid & 31) == 0) red[tid >> 5] = v;
    named_bar_sync(1 + group, RT);
    v = 0.f;
#pragma unroll
    for (int k = 0; k < RT / 32; ++k) v += red[k];
  }
  return v;
}

// Which of the eight elements of block `block` are kept.  limit = (threshold << 16) - 1: 16 bits
// u are >= threshold where (u << 16) > limit; the bits below do not matter for the upper half of
// a word, which is compared as it is.
struct Keep {
  uint32_t w[4];
  uint32_t limit;
  __device__ __forceinline__ void draw(const DropArgs& d, uint64_t seed, uint64_t block) {
    const uint4 r = philox_block(block, d.stream, seed);
    w[0] = r.x;
    w[1] = r.y;
    w[2] = r.z;
    w[3] = r.w;
    limit = (static_cast<uint32_t>(d.threshold) << 16) - 1u;
  }
  // zero, not a product, where dropped: what is there need not be finite
  __device__ __forceinline__ void apply(float2* v) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j].x = (w[j] << 16) > limit ? v[j].x : 0.f;
      v[j].y = w[j] > limit ? v[j].y : 0.f;
    }
  }
};
__device__ __forceinline__ uint64_t seed_of(const DropArgs& d) {
  return d.seed_ptr != nullptr ? static_cast<uint64_t>(*d.seed_ptr) : d.seed;
}

// The columns of a thread.  Every thread takes NV blocks of eight elements that begin on
// multiples of eight of the tensor's flat index.  Where the width is not a multiple of eight (ODD)
// a row starts `shift` elements into its first block, and blocks at a row's ends are partial; a
// group's rows are eight apart (or a multiple), so its shift and its threads' columns stay.
template <typename T, int NV, int RT, bool ODD>
struct Cols {
  int H, tid, shift;
  int64_t total;
  __device__ __forceinline__ Cols(const JoinArgs& a, int tid_, int64_t row0)
      : H(a.H), tid(tid_), shift(ODD ? static_cast<int>((row0 * a.H) & 7) : 0), total(a.T * a.H) {}
  __device__ __forceinline__ int col(int k) const { return (tid + k * RT) * 8 - shift; }
  __device__ __forceinline__ bool on(int k) const { return col(k) < H; }
  __device__ __forceinline__ bool whole(int k) const {
    return !ODD || (col(k) >= 0 && col(k) + 8 <= H);
  }
  // 0 in the elements of a partial block that are the neighbouring rows'
  __device__ __forceinline__ void clear(Oct<T>& o, int k) const {
    const int c = col(k);
    T* e = reinterpret_cast<T*>(o.raw);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < 0 || c + j >= H) e[j] = from_f<T>(0.f);
  }
  __device__ __forceinline__ void load(Oct<T>& o, const T* p, int64_t base, int k) const {
    if (whole(k)) {
      o.load_once(p + base + col(k));
    } else {
      const int c = col(k);
      T* e = reinterpret_cast<T*>(o.raw);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        e[j] = c + j >= 0 && c + j < H ? p[base + c + j] : from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ void store(T* p, int64_t base, int k, const float2* v) const {
    if (whole(k)) {
      Oct<T>::store(p + base + col(k), v);
    } else {
      const int c = col(k);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c + 2 * j >= 0 && c + 2 * j < H) p[base + c + 2 * j] = from_f<T>(v[j].x);
        if (c + 2 * j + 1 >= 0 && c + 2 * j + 1 < H) p[base + c + 2 * j + 1] = from_f<T>(v[j].y);
      }
    }
  }
  // a weight's columns, times v
  __device__ __forceinline__ void times(const T* w, int k, float2* v) const {
    if (!ODD) {
      Oct<T> o;
      float2 u[4];
      o.load(w + col(k));
      o.get(u);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = mul2(v[j], u[j]);
    } else {
      const int c = col(k);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c + 2 * j >= 0 && c + 2 * j < H) v[j].x *= to_f<T>(w[c + 2 * j]);
        if (c + 2 * j + 1 >= 0 && c + 2 * j + 1 < H) v[j].y *= to_f<T>(w[c + 2 * j + 1]);
      }
    }
  }
  // f * w1 * gate, the branch's factors (null: 1)
  __device__ __forceinline__ void factors(const JoinArgs& a, float f, int k, float2* v) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = splat(f);
    if (a.w1 != nullptr) times(static_cast<const T*>(a.w1), k, v);
    if (a.gate != nullptr) times(static_cast<const T*>(a.gate), k, v);
  }
};

// The input rows of a group.  With RING they come through shared memory: one thread keeps
// `stages` rows of bulk copies in flight, whatever the threads compute meanwhile, and nothing of a
// row has to stay in registers from one of its sums to the next.  Without, a row is loaded into
// registers (rows so wide that two do not fit).  A copy takes the row's whole blocks, which start
// on 16-byte boundaries also where the row does not (the tensor's last block, where it is not
// whole, is left out); a row's partial blocks are put right by the threads that read them.  A wait
// that runs out is reported and the rows that follow are computed from what is there.
template <typename T, int NV, int RT, int NT, bool ODD, bool RING, bool FULL>
struct Feed {
  const T* p[NT];  // null: not read (none with FULL)
  Oct<T> reg[RING ? 1 : NT][RING ? 1 : NV];
  const Cols<T, NV, RT, ODD>& cols;
  uint8_t* ring;
  uint64_t* bar;
  volatile int* abort_flag;
  int* err;
  int stages, stage, row_bytes, group;
  uint32_t phase;
  int64_t step, T_rows, issued, base;

  __device__ __forceinline__ Feed(const JoinArgs& a, const Cols<T, NV, RT, ODD>& c, uint8_t* smem,
                                  uint64_t* bars, int* flag, int stages_, int group_, int64_t step_)
      : cols(c), ring(smem), bar(bars), abort_flag(flag), err(a.err), stages(stages_), stage(0),
        row_bytes(pitch(a.H) * static_cast<int>(sizeof(T))), group(group_), phase(0), step(step_),
        T_rows(a.T), issued(0), base(0) {}
  static __host__ __device__ constexpr int pitch(int H) { return ODD ? (H + 14) / 8 * 8 : H; }
  __device__ __forceinline__ uint8_t* at(int s, int i) const {
    return ring + (static_cast<int64_t>(s) * NT + i) * row_bytes;
  }
  __device__ __forceinline__ void issue(int s, int64_t row) {
    ++issued;
    int n = 0;
#pragma unroll
    for (int i = 0; i < NT; ++i) n += FULL || p[i] != nullptr ? 1 : 0;
    const int64_t first = row * cols.H - cols.shift;
    uint32_t bytes = static_cast<uint32_t>(row_bytes);
    if constexpr (ODD) {
      int64_t blocks = (cols.H + cols.shift + 7) / 8;
      const int64_t most = (cols.total - first) / 8;
      if (blocks > most) blocks = most;
      bytes = static_cast<uint32_t>(blocks * 8 * static_cast<int>(sizeof(T)));
    }
    mbar_arrive_expect_tx(&bar[s], n * bytes);
    if (bytes == 0) return;
#pragma unroll
    for (int i = 0; i < NT; ++i)
      if (FULL || p[i] != nullptr) bulk_load(at(s, i), p[i] + first, bytes, &bar[s]);
  }
  __device__ __forceinline__ void start(int64_t row0) {
    if constexpr (RING) {
      if (cols.tid == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(&bar[s], 1);
        fence_barrier_init();
        fence_proxy_async_shared();
        for (int s = 0; s < stages; ++s)
          if (row0 + s * step < T_rows) issue(s, row0 + s * step);
      }
      sync();
    }
  }
  __device__ __forceinline__ void sync() const {
    if constexpr (RT > 32)
      named_bar_sync(1 + group, RT);
    else
      __syncwarp();
  }
  __device__ __forceinline__ void begin(int64_t row) {
    base = row * cols.H;
    if constexpr (RING) {
      mbar_wait(&bar[stage], phase, abort_flag, err, kErrTimeoutFull, 61);
      if constexpr (ODD) {  // blocks at the row's ends, each read by this thread alone
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if (cols.on(k) && !cols.whole(k)) {
            const bool copied = base + cols.col(k) + 8 <= cols.total;
#pragma unroll
            for (int i = 0; i < NT; ++i)
              if (FULL || p[i] != nullptr) {
                uint4* q = reinterpret_cast<uint4*>(at(stage, i)) +
                           (cols.tid + k * RT) * static_cast<int>(sizeof(T) / 2);
                Oct<T> o;
                if (copied) {
#pragma unroll
                  for (int w = 0; w < static_cast<int>(sizeof(T) / 2); ++w) o.raw[w] = q[w];
                  cols.clear(o, k);
                } else {
                  cols.load(o, p[i], base, k);
                }
#pragma unroll
                for (int w = 0; w < static_cast<int>(sizeof(T) / 2); ++w) q[w] = o.raw[w];
              }
            fence_proxy_async_shared();  // before the stage's next copy
          }
      }
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (cols.on(k)) {
#pragma unroll
          for (int i = 0; i < NT; ++i)
            if (FULL || p[i] != nullptr) cols.load(reg[i][k], p[i], row * cols.H, k);
        }
    }
  }
  __device__ __forceinline__ void get(int i, int k, float2* v) const {
    if constexpr (RING) {
      Oct<T> o;
      const uint4* q = reinterpret_cast<const uint4*>(at(stage, i)) +
                       (cols.tid + k * RT) * static_cast<int>(sizeof(T) / 2);
#pragma unroll
      for (int j = 0; j < static_cast<int>(sizeof(T) / 2); ++j) o.raw[j] = q[j];
      o.get(v);
    } else {
      reg[i][k].get(v);
    }
  }
  // Every thread is done with the row (the barrier also keeps a sum's slots of two rows apart); its
  // stage takes the row `stages` further on.  Refilling it only after the next row's first sum
  // would save the barrier, and measured slower (backward of 32768 x 896: 92 -> 103 us).
  __device__ __forceinline__ void end(int64_t row) {
    sync();
    if constexpr (RING) {
      if (cols.tid == 0 && row + stages * step < T_rows && *abort_flag == 0)
        issue(stage, row + stages * step);
      if (++stage == stages) {
        stage = 0;
        phase ^= 1;
      }
    }
  }
  // after a wait that ran out: a bounded wait for the copies that are still under way
  __device__ __forceinline__ void drain() {
    if constexpr (RING) {
      if (*abort_flag != 0 && cols.tid == 0)
        for (int s = 0; s < stages && s < issued; ++s)
          mbar_wait(&bar[s], static_cast<uint32_t>(((issued - 1 - s) / stages) & 1), nullptr, err,
                    kErrTimeoutFull, 62);
    }
  }
};

// CTAs an SM that a kernel's registers have to allow.  Odd widths' conditions would otherwise take
// a fifth warp's registers: 20000 x 1111 with dropout, forward 121 us without the bound, 83 with
// four CTAs, backward 149 and 121 with three; three for the smallest rows' backward spills.
__host__ __device__ constexpr int ctas_of(int nv, int rt, int most) {
  return rt == 512 ? 1 : nv == 1 && rt == 256 ? most : 2;
}

// The branch's factors f * w1 * gate and the norm's weights w2 (1 where there are none) of a
// thread's columns: in registers for all rows (up to two blocks a thread), in shared memory as
// fp32 (a warp a row: its four blocks would take 64 registers), or read again from L1 for every
// row (four blocks of the widest rows).
enum Hold { kInRegs, kInShared, kAgain };
__host__ __device__ constexpr Hold hold_of(int nv, int rt) {
  return nv <= 2 ? kInRegs : rt == 32 ? kInShared : kAgain;
}

template <typename T, int NV, int RT, bool ODD>
struct Weights {
  static constexpr Hold how = hold_of(NV, RT);
  const JoinArgs& a;
  const Cols<T, NV, RT, ODD>& cols;
  const float f;
  float2 c[how == kInRegs ? NV : 1][4], v2[how == kInRegs ? NV : 1][4];
  float4* shared;  // [4][H / 8]: lower and upper halves of the factors, of w2

  __device__ __forceinline__ Weights(const JoinArgs& a_, const Cols<T, NV, RT, ODD>& cols_, float f_,
                                     void* smem)
      : a(a_), cols(cols_), f(f_), shared(static_cast<float4*>(smem)) {
    if constexpr (how == kInRegs) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (cols.on(k)) {
          cols.factors(a, f, k, c[k]);
          norm_from(k, v2[k]);
        }
    } else if constexpr (how == kInShared) {
      const int n8 = a.H / 8;
      for (int i = threadIdx.x; i < 4 * n8; i += blockDim.x) {
        float* out = reinterpret_cast<float*>(shared + i);
        const int o = i % n8, c0 = o * 8 + (i / n8 & 1) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v = 1.f;
          if (i / n8 < 2) {
            v = f;
            if (a.w1 != nullptr) v *= to_f<T>(static_cast<const T*>(a.w1)[c0 + j]);
            if (a.gate != nullptr) v *= to_f<T>(static_cast<const T*>(a.gate)[c0 + j]);
          } else if (a.w2 != nullptr) {
            v = to_f<T>(static_cast<const T*>(a.w2)[c0 + j]);
          }
          out[j] = v;
        }
      }
      __syncthreads();
    }
  }
  __device__ __forceinline__ void norm_from(int k, float2* t) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = splat(1.f);
    if (a.w2 != nullptr) cols.times(static_cast<const T*>(a.w2), k, t);
  }
  __device__ __forceinline__ void from_shared(int which, int k, float2* t) const {
    const int n8 = a.H / 8, o = cols.tid + k * RT;
    const float4 lo = shared[2 * which * n8 + o], hi = shared[(2 * which + 1) * n8 + o];
    t[0] = make_float2(lo.x, lo.y);
    t[1] = make_float2(lo.z, lo.w);
    t[2] = make_float2(hi.x, hi.y);
    t[3] = make_float2(hi.z, hi.w);
  }
  __device__ __forceinline__ void branch(int k, float2* t) const {
    if constexpr (how == kInRegs) {
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = c[k][j];
    } else if constexpr (how == kInShared) {
      from_shared(0, k, t);
    } else {
      cols.factors(a, f, k, t);
    }
  }
  __device__ __forceinline__ void norm(int k, float2* t) const {
    if constexpr (how == kInRegs) {
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = v2[k][j];
    } else if constexpr (how == kInShared) {
      from_shared(1, k, t);
    } else {
      norm_from(k, t);
    }
  }
};

template <typename T, int NV, int RT, bool ODD, bool DROP, bool RING, bool FULL>
__global__ void __launch_bounds__(RT > 256 ? RT : 256, ctas_of(NV, RT, 4))
    join_fwd_k(const JoinArgs a, float factor, int stages) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t bars[8][kMaxStages];
  __shared__ int abort_flag;
  __shared__ float red_all[2][32];
  const int group = threadIdx.x / RT, tid = threadIdx.x % RT, groups = blockDim.x / RT;
  float* red0 = red_all[0] + group * (RT / 32);
  float* red1 = red_all[1] + group * (RT / 32);
  const bool post = FULL || a.w1 != nullptr, norm = FULL || a.w2 != nullptr;
  const uint64_t seed = DROP ? seed_of(a.drop) : 0;
  const float inv_h = 1.f / a.H, f = a.scale * factor;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * groups + group;
  const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
  const Cols<T, NV, RT, ODD> cols(a, tid, row0);
  if (threadIdx.x == 0) abort_flag = 0;
  __syncthreads();
  using In = Feed<T, NV, RT, 2, ODD, RING, FULL>;
  const int ring_bytes = stages * 2 * In::pitch(a.H) * static_cast<int>(sizeof(T));  // of a group
  In in(a, cols, ring + group * ring_bytes, bars[group], &abort_flag, stages, group, step);
  in.p[0] = static_cast<const T*>(a.x);
  in.p[1] = static_cast<const T*>(a.b);
  in.start(row0);
  const Weights<T, NV, RT, ODD> weights(a, cols, f, ring + groups * ring_bytes);
  for (int64_t row = row0; row < a.T; row += step) {
    const int64_t base = row * a.H;
    in.begin(row);
    float r1 = 1.f;
    if (post) {
      float2 ss = splat(0.f);
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (cols.on(k)) {
          float2 v[4];
          in.get(1, k, v);
#pragma unroll
          for (int j = 0; j < 4; ++j) ss = fma2(v[j], v[j], ss);
        }
      r1 = rsqrtf(row_sum<RT>(ss.x + ss.y, red0, group, tid) * inv_h + a.eps);
      if (a.r1 != nullptr && tid == 0) a.r1[row] = r1;
    }
    float2 nx[NV][4];
    float2 ss = splat(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (cols.on(k)) {
        float2 u[4];
        in.get(1, k, u);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = mul2(u[j], splat(r1));
        if constexpr (DROP) {
          Keep m;
          m.draw(a.drop, seed, static_cast<uint64_t>(base + cols.col(k)) >> 3);
          m.apply(u);
        }
        in.get(0, k, nx[k]);
        float2 t[4];
        weights.branch(k, t);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          nx[k][j] = fma2(u[j], t[j], nx[k][j]);
          ss = fma2(nx[k][j], nx[k][j], ss);
        }
        cols.store(static_cast<T*>(a.xnew), base, k, nx[k]);
      }
    if (norm) {
      // from x' in 32 bits: y carries one rounding, its own
      const float r2 = rsqrtf(row_sum<RT>(ss.x + ss.y, red1, group, tid) * inv_h + a.eps);
      if (a.r2 != nullptr && tid == 0) a.r2[row] = r2;
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (cols.on(k)) {
          float2 t[4];
          weights.norm(k, t);
#pragma unroll
          for (int j = 0; j < 4; ++j) nx[k][j] = mul2(mul2(nx[k][j], splat(r2)), t[j]);
          cols.store(static_cast<T*>(a.y), base, k, nx[k]);
        }
    }
    in.end(row);
  }
  in.drain();
}

template <typename T, int NV, int RT, bool ODD, bool DROP, bool RING, bool FULL>
__global__ void __launch_bounds__(RT > 256 ? RT : 256, ctas_of(NV, RT, 3))
    join_bwd_k(const JoinArgs a, float factor, int stages) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t bars[8][kMaxStages];
  __shared__ int abort_flag;
  __shared__ float red_all[2][32];
  const int group = threadIdx.x / RT, tid = threadIdx.x % RT, groups = blockDim.x / RT;
  float* red0 = red_all[0] + group * (RT / 32);
  float* red1 = red_all[1] + group * (RT / 32);
  const T* dxn = static_cast<const T*>(a.dxnew);
  const T* dy = static_cast<const T*>(a.dy);
  const uint64_t seed = DROP ? seed_of(a.drop) : 0;
  const float inv_h = 1.f / a.H, f = a.scale * factor;
  const bool post = FULL || a.w1 != nullptr;
  const bool has_dy = FULL || dy != nullptr, has_dxn = FULL || dxn != nullptr;
  const bool branch = FULL || a.db != nullptr || a.dgate != nullptr || a.dw1 != nullptr;
  // b itself enters the gradients
  const bool need_b = FULL || (branch && (post || a.dgate != nullptr));
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * groups + group;
  const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
  const Cols<T, NV, RT, ODD> cols(a, tid, row0);
  if (threadIdx.x == 0) abort_flag = 0;
  __syncthreads();
  using In = Feed<T, NV, RT, 4, ODD, RING, FULL>;
  const int ring_bytes = stages * 4 * In::pitch(a.H) * static_cast<int>(sizeof(T));  // of a group
  In in(a, cols, ring + group * ring_bytes, bars[group], &abort_flag, stages, group, step);
  in.p[0] = dy;
  in.p[1] = has_dy ? static_cast<const T*>(a.xnew) : nullptr;
  in.p[2] = dxn;
  in.p[3] = need_b ? static_cast<const T*>(a.b) : nullptr;
  in.start(row0);
  const Weights<T, NV, RT, ODD> weights(a, cols, f, ring + groups * ring_bytes);
  float2 s1[NV][4], s2[NV][4];  // columns' sums of g m bh and dy xh
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) s1[k][j] = s2[k][j] = splat(0.f);
  float r1_next = 1.f, r2_next = 0.f;
  if (row0 < a.T) {
    if (FULL || a.r1 != nullptr) r1_next = a.r1[row0];
    if (has_dy) r2_next = a.r2[row0];
  }
  for (int64_t row = row0; row < a.T; row += step) {
    const int64_t base = row * a.H;
    in.begin(row);
    // the next row's statistics are on their way while this one is computed
    const float r1 = r1_next, r2 = r2_next;
    if (row + step < a.T) {
      if (FULL || a.r1 != nullptr) r1_next = a.r1[row + step];
      if (has_dy) r2_next = a.r2[row + step];
    }
    float mean = 0.f;
    if (has_dy) {
      float2 dot = splat(0.f);
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (cols.on(k)) {
          float2 d[4], v[4];
          in.get(0, k, d);
          in.get(1, k, v);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            d[j] = mul2(d[j], mul2(v[j], splat(r2)));
            s2[k][j] = add2(s2[k][j], d[j]);
          }
          weights.norm(k, v);
#pragma unroll
          for (int j = 0; j < 4; ++j) dot = fma2(d[j], v[j], dot);
        }
      mean = row_sum<RT>(dot.x + dot.y, red0, group, tid) * inv_h;
    }
    float2 g[NV][4];
    float2 dot = splat(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (cols.on(k)) {
        if (has_dxn) {
          in.get(2, k, g[k]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) g[k][j] = splat(0.f);
        }
        if (has_dy) {
          float2 d[4], v[4], t[4];
          in.get(0, k, d);
          in.get(1, k, v);
          weights.norm(k, t);
          const float2 sub = splat(-r2 * r2 * mean);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            g[k][j] = fma2(mul2(d[j], t[j]), splat(r2), g[k][j]);
            g[k][j] = fma2(v[j], sub, g[k][j]);
          }
        }
        if (FULL || a.dx != nullptr) cols.store(static_cast<T*>(a.dx), base, k, g[k]);
        if (branch) {
          float2 bh[4], t[4];
          Keep m;
          if constexpr (DROP) {
            m.draw(a.drop, seed, static_cast<uint64_t>(base + cols.col(k)) >> 3);
            m.apply(g[k]);
          }
          if (need_b) {
            in.get(3, k, bh);
            // with its norm a branch that is not finite makes the whole row so
            if (DROP && !post) m.apply(bh);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              bh[j] = mul2(bh[j], splat(r1));
              s1[k][j] = fma2(g[k][j], bh[j], s1[k][j]);
            }
          }
          weights.branch(k, t);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            g[k][j] = mul2(g[k][j], t[j]);
            if (post) dot = fma2(g[k][j], bh[j], dot);
          }
        }
      }
    if (branch) {
      if (post) {
        const float2 sub =
            splat(-r1 * r1 * (row_sum<RT>(dot.x + dot.y, red1, group, tid) * inv_h));
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if (cols.on(k)) {
            float2 v[4];
            in.get(3, k, v);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              g[k][j] = fma2(v[j], sub, mul2(g[k][j], splat(r1)));
          }
      }
      if (FULL || a.db != nullptr) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if (cols.on(k)) cols.store(static_cast<T*>(a.db), base, k, g[k]);
      }
    }
    in.end(row);
  }
  in.drain();
  if (a.partials == nullptr) return;
  grid_dependents_go();
  // the groups of the CTA one after the other, through this CTA's part of the workspace
  float* p = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * a.H;
  for (int q = 0; q < groups; ++q) {
    if (q == group) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c0 = cols.col(k);
        const float* u1 = reinterpret_cast<const float*>(s1[k]);
        const float* u2 = reinterpret_cast<const float*>(s2[k]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c0 + j >= 0 && c0 + j < a.H) {
            float* at = p + c0 + j;
            at[0] = (q == 0 ? 0.f : at[0]) + u1[j];
            at[a.H] = (q == 0 ? 0.f : at[a.H]) + u2[j];
          }
      }
    }
    __syncthreads();
  }
}

// The CTAs' column sums, 32 columns a block, 32 threads a column, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) join_cols_k(const JoinArgs a, int blocks, float f) {
  __shared__ float t1[32][33], t2[32][33];
  grid_dependency_wait();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  float s1 = 0.f, s2 = 0.f;
  if (c < a.H) {
#pragma unroll 4
    for (int i = ty; i < blocks; i += 32) {
      const float* p = a.partials + static_cast<int64_t>(i) * 2 * a.H + c;
      s1 += p[0];
      s2 += p[a.H];
    }
  }
  t1[ty][tx] = s1;
  t2[ty][tx] = s2;
  __syncthreads();
  s1 = f * warp_sum(t1[tx][ty]);
  s2 = warp_sum(t2[tx][ty]);
  const int col = blockIdx.x * 32 + ty;
  if (tx != 0 || col >= a.H) return;
  const T* w1 = static_cast<const T*>(a.w1);
  const T* gate = static_cast<const T*>(a.gate);
  if (a.dw2 != nullptr) static_cast<T*>(a.dw2)[col] = from_f<T>(s2);
  if (a.dgate != nullptr)
    static_cast<T*>(a.dgate)[col] = from_f<T>(w1 != nullptr ? s1 * to_f<T>(w1[col]) : s1);
  if (a.dw1 != nullptr)
    static_cast<T*>(a.dw1)[col] = from_f<T>(gate != nullptr ? s1 * to_f<T>(gate[col]) : s1);
}

// y = m * x / kept share: kDropVecs blocks of eight elements a thread, loaded before the generator
// runs for them (one a turn of a persistent grid: 31 us where four take 21, 32768 x 896 bf16).
constexpr int kDropVecs = 4;

template <typename T>
__global__ void __launch_bounds__(256) dropout_k(const T* __restrict__ x, T* __restrict__ y,
                                                 int64_t n, const DropArgs d, float factor) {
  const uint64_t seed = seed_of(d);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 256 * kDropVecs + threadIdx.x;
  Oct<T> in[kDropVecs];
#pragma unroll
  for (int k = 0; k < kDropVecs; ++k) {
    const int64_t e = (first + k * 256) * 8;
    if (e + 8 <= n) in[k].load_once(x + e);
  }
#pragma unroll
  for (int k = 0; k < kDropVecs; ++k) {
    const int64_t e = (first + k * 256) * 8;
    if (e >= n) break;
    Keep m;
    float2 v[4];
    m.draw(d, seed, static_cast<uint64_t>(e) >> 3);
    if (e + 8 <= n) {
      in[k].get(v);
      m.apply(v);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = mul2(v[j], splat(factor));
      Oct<T>::store(y + e, v);
    } else {
      float* s = reinterpret_cast<float*>(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = e + j < n ? to_f<T>(x[e + j]) : 0.f;
      m.apply(v);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e + j < n) y[e + j] = from_f<T>(s[j] * factor);
    }
  }
}

// ---------------------------------------------------------------- host side
// Calls f with the (NV, RT, ODD) of a row: the fewest threads that hold it.  Up to 128 blocks of a
// 16-bit type, with rows for every warp of the machine, take fewer threads with more blocks each:
// a row's fixed work (its sums and barriers) is then one or two warps' instead of four's.  32768 x
// 896 with dropout, us, before what `full` saves: forward 60 with four warps a row, 51 with one;
// backward 123 with four, 114 with two (one: 153, its columns' sums leave 8 warps an SM).
template <typename T, bool BWD, typename F>
int with_shape(const JoinArgs& a, int num_sms, F f) {
  const bool odd = a.H % 8 != 0;
  const int n = odd ? (a.H + 14) / 8 : a.H / 8;
  const auto go = [&](auto nv, auto rt) {
    return odd ? f(nv, rt, std::true_type()) : f(nv, rt, std::false_type());
  };
  using std::integral_constant;
  if (n <= 32) return go(integral_constant<int, 1>(), integral_constant<int, 32>());
  if constexpr (sizeof(T) == 2) {
    if (n <= 128 && a.T >= 16 * num_sms) {
      if constexpr (!BWD)
        if (!odd)
          return f(integral_constant<int, 4>(), integral_constant<int, 32>(), std::false_type());
      return go(integral_constant<int, 2>(), integral_constant<int, 64>());
    }
  }
  if (n <= 128) return go(integral_constant<int, 1>(), integral_constant<int, 128>());
  if (n <= 256) return go(integral_constant<int, 1>(), integral_constant<int, 256>());
  if (n <= 512) return go(integral_constant<int, 2>(), integral_constant<int, 256>());
  if (n <= 1024) return go(integral_constant<int, 2>(), integral_constant<int, 512>());
  if (n <= 2048) return go(integral_constant<int, 4>(), integral_constant<int, 512>());
  return -2;
}

// Rows side by side in a CTA: as many as fill 256 threads, fewer where that leaves SMs idle.
inline int groups_of(int rt, int64_t rows, int num_sms) {
  int g = rt >= 256 ? 1 : 256 / rt;
  while (g > 1 && (rows + g - 1) / g < num_sms) g /= 2;
  return g;
}

// A launch: shared memory of the rings and the CTAs of the persistent grid.
struct JoinLaunch {
  int groups = 1, threads = 0, stages = 0, smem = 0, grid = 1;
};

// Stages of a group's ring: the CTA's share of an SM's shared memory where the SM holds 768
// threads (512 with two blocks a thread, which take more registers); all of it where the share is
// less than two rows; 0, no ring, where that is too.
inline int ring_stages(const JoinArgs& a, int tensors, int groups, int rt, int nv) {
  const int64_t row = static_cast<int64_t>(a.H % 8 == 0 ? a.H : (a.H + 14) / 8 * 8) *
                      (a.type == kStreamFloat ? 4 : 2) * tensors * groups;
  const int64_t whole = 220 * 1024, share = whole * (rt * groups) / (nv == 1 ? 768 : 512);
  int64_t n = share / row;
  if (n < 2) n = whole / row;
  return n < 2 ? 0 : n > kMaxStages ? kMaxStages : static_cast<int>(n);
}

// One CTA for each `groups` rows, at most what is resident at once; a group's rows are a multiple
// of eight apart where the width is not a multiple of eight.
template <typename K>
int grid_of(K kern, const JoinLaunch& l, const JoinArgs& a, int num_sms) {
  const int64_t want = a.T > 0 ? (a.T + l.groups - 1) / l.groups : 1;
  int64_t grid = want;
  if (want > num_sms) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, l.threads, l.smem) !=
            cudaSuccess || n < 1)
      n = 1;
    const int64_t most = static_cast<int64_t>(num_sms) * n;
    if (most < grid) grid = most;
  }
  if (a.H % 8 != 0) grid = grid < 8 ? 8 : grid / 8 * 8;
  return static_cast<int>(grid);
}

}  // namespace

// Calls f(kernel, launch) with the kernel of a call's width, norms and dropout.
template <typename T, bool BWD, typename F>
static int with_kernel(const JoinArgs& a, int num_sms, F f) {
  return with_shape<T, BWD>(a, num_sms, [&](auto nv, auto rt, auto odd) {
    constexpr int NV = decltype(nv)::value, RT = decltype(rt)::value;
    constexpr bool ODD = decltype(odd)::value;
    JoinLaunch l;
    l.groups = groups_of(RT, a.T, num_sms);
    l.threads = RT * l.groups;
    constexpr int tensors = BWD ? 4 : 2;
    l.stages = ring_stages(a, tensors, l.groups, RT, NV);
    l.smem = l.stages * l.groups * tensors *
             Feed<T, NV, RT, tensors, ODD, true, true>::pitch(a.H) * static_cast<int>(sizeof(T));
    if (hold_of(NV, RT) == kInShared) l.smem += 8 * a.H;
    const auto go = [&](auto kern) {
      if (l.smem > 40 * 1024) {  // up to 48 KB with the static part need no consent
        // one value for every call: another thread's smaller one must not undo this one's
        const cudaError_t e = cudaFuncSetAttribute(
            kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if (e != cudaSuccess) return static_cast<int>(e);
      }
      l.grid = grid_of(kern, l, a, num_sms);
      return f(kern, l);
    };
    // Every norm there and every gradient wanted: kernels without the questions, which a row
    // asks some twenty times (backward of 32768 x 896: 93 us with them, 75 without).
    const bool full = a.w1 != nullptr && a.w2 != nullptr &&
                      (!BWD || (a.dy != nullptr && a.dxnew != nullptr && a.dx != nullptr &&
                                a.db != nullptr));
    const auto pick = [&](auto drop, auto ring, auto all) {
      constexpr bool D = decltype(drop)::value, R = decltype(ring)::value,
                     A = decltype(all)::value;
      if constexpr (BWD)
        return go(join_bwd_k<T, NV, RT, ODD, D, R, A>);
      else
        return go(join_fwd_k<T, NV, RT, ODD, D, R, A>);
    };
    const auto pick_full = [&](auto drop, auto ring) {
      return full ? pick(drop, ring, std::true_type()) : pick(drop, ring, std::false_type());
    };
    if (l.stages > 0)
      return a.drop.threshold > 0 ? pick_full(std::true_type(), std::true_type())
                                  : pick_full(std::false_type(), std::true_type());
    if constexpr (RT == 512)  // the widest rows alone can be without a ring
      return a.drop.threshold > 0 ? pick(std::true_type(), std::false_type(), std::false_type())
                                  : pick(std::false_type(), std::false_type(), std::false_type());
    return -2;
  });
}

template <typename T>
int join_fwd_t(const JoinArgs& a, int num_sms, cudaStream_t s) {
  return with_kernel<T, false>(a, num_sms, [&](auto kern, const JoinLaunch& l) {
    kern<<<l.grid, l.threads, l.smem, s>>>(a, a.drop.factor(), l.stages);
    return static_cast<int>(cudaGetLastError());
  });
}

template <typename T>
int join_bwd_blocks_t(const JoinArgs& a, int num_sms) {
  int blocks = -1;
  const int rc = with_kernel<T, true>(a, num_sms, [&](auto, const JoinLaunch& l) {
    blocks = l.grid;
    return 0;
  });
  return rc != 0 ? -1 : blocks;
}

template <typename T>
int join_bwd_t(const JoinArgs& a, int num_sms, cudaStream_t s) {
  return with_kernel<T, true>(a, num_sms, [&](auto kern, const JoinLaunch& l) {
    kern<<<l.grid, l.threads, l.smem, s>>>(a, a.drop.factor(), l.stages);
    const int rc = static_cast<int>(cudaGetLastError());
    if (rc != 0 || a.partials == nullptr) return rc;
    return launch_dependent(join_cols_k<T>, dim3((a.H + 31) / 32), 1024, s, a, l.grid,
                            a.scale * a.drop.factor());
  });
}

template <typename T>
int dropout_t(const void* x, void* y, int64_t n, const DropArgs& d, cudaStream_t s) {
  const int64_t each = static_cast<int64_t>(256) * 8 * kDropVecs;
  if ((n + each - 1) / each > 0x7fffffff) return -2;
  if (d.threshold == 0)
    return static_cast<int>(cudaMemcpyAsync(y, x, n * sizeof(T), cudaMemcpyDeviceToDevice, s));
  dropout_k<T><<<static_cast<unsigned>((n + each - 1) / each), 256, 0, s>>>(
      static_cast<const T*>(x), static_cast<T*>(y), n, d, d.factor());
  return static_cast<int>(cudaGetLastError());
}

#define CFB_STREAM_TYPE(T)                                                                \
  template int join_fwd_t<T>(const JoinArgs&, int, cudaStream_t);                         \
  template int join_bwd_blocks_t<T>(const JoinArgs&, int);                                \
  template int join_bwd_t<T>(const JoinArgs&, int, cudaStream_t);                         \
  template int dropout_t<T>(const void*, void*, int64_t, const DropArgs&, cudaStream_t);

}  // namespace cfb
