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
// All of it is bound by memory.  The forward reads x, b and writes x', y; the backward reads dx',
// dy, x', b and writes dx, db; the dropout mask is drawn again from its counter instead of being
// stored.  A row lies in the registers of RT threads; sums run in fp32; results are rounded once,
// at their stores.  The columns' sums stay in registers over all rows of a CTA, and one small
// kernel adds the CTAs' sums in a fixed order, so that equal calls give equal bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

// VEC elements: one 16-byte access, or one element where rows are not in 16-byte units.
template <typename T, int VEC>
struct Vec {
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void load_once(const T* p) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w)
                 : "l"(p));
  }
  __device__ __forceinline__ void get(float* v) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = to_f<T>(e[j]);
  }
  static __device__ __forceinline__ void store(T* p, const float* v) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = from_f<T>(v[j]);
    *reinterpret_cast<uint4*>(p) = u;
  }
};
template <typename T>
struct Vec<T, 1> {
  T raw;
  __device__ __forceinline__ void load(const T* p) { raw = *p; }
  __device__ __forceinline__ void load_once(const T* p) { raw = *p; }
  __device__ __forceinline__ void get(float* v) const { v[0] = to_f<T>(raw); }
  static __device__ __forceinline__ void store(T* p, const float* v) { *p = from_f<T>(v[0]); }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the RT threads of a row.  `red` holds RT / 32 floats of this row's group; the caller
// alternates between two of them, so one barrier a sum is enough.
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

// Dropout factors of VEC elements from element e on (a multiple of VEC).
template <int VEC>
__device__ __forceinline__ void drop_factors(const DropArgs& d, uint64_t seed, float factor,
                                             int64_t e, float* m) {
  const uint4 r = philox_block(static_cast<uint64_t>(e) >> 3, d.stream, seed);
  if constexpr (VEC == 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = philox_lane(r, j) >= d.threshold ? factor : 0.f;
  } else if constexpr (VEC == 4) {
    const bool high = (e & 4) != 0;
    const uint4 h = make_uint4(high ? r.z : r.x, high ? r.w : r.y, 0u, 0u);
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = philox_lane(h, j) >= d.threshold ? factor : 0.f;
  } else {
    const int j = static_cast<int>(e & 7);
    const uint32_t w = j < 4 ? (j < 2 ? r.x : r.y) : (j < 6 ? r.z : r.w);
    const int u = static_cast<int>((j & 1) ? w >> 16 : w & 0xffffu);
    m[0] = u >= d.threshold ? factor : 0.f;
  }
}

// A dropped element is 0 whatever it was (not 0 * NaN).
__device__ __forceinline__ float masked(float v, float m) { return m == 0.f ? 0.f : v * m; }

template <typename T, int VEC, int NV, int RT, bool DROP>
__global__ void __launch_bounds__(RT > 256 ? RT : 256)
    join_fwd_k(const JoinArgs a, float factor) {
  __shared__ float red_all[2][32];
  const int group = threadIdx.x / RT, tid = threadIdx.x % RT, groups = blockDim.x / RT;
  float* red0 = red_all[0] + group * (RT / 32);
  float* red1 = red_all[1] + group * (RT / 32);
  const int nv = a.H / VEC;
  const T* x = static_cast<const T*>(a.x);
  const T* b = static_cast<const T*>(a.b);
  const T* w1 = static_cast<const T*>(a.w1);
  const T* gate = static_cast<const T*>(a.gate);
  const T* w2 = static_cast<const T*>(a.w2);
  uint64_t seed = 0;
  if constexpr (DROP)
    seed = a.drop.seed_ptr != nullptr ? static_cast<uint64_t>(*a.drop.seed_ptr) : a.drop.seed;
  const float inv_h = 1.f / a.H;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * groups + group; row < a.T;
       row += static_cast<int64_t>(gridDim.x) * groups) {
    const int64_t base = row * a.H;
    Vec<T, VEC> bv[NV], xv[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = tid + k * RT;
      if (i < nv) {
        bv[k].load_once(b + base + static_cast<int64_t>(i) * VEC);
        xv[k].load_once(x + base + static_cast<int64_t>(i) * VEC);
      }
    }
    float r1 = 1.f;
    if (w1 != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (tid + k * RT < nv) {
          float v[VEC];
          bv[k].get(v);
#pragma unroll
          for (int j = 0; j < VEC; ++j) ss += v[j] * v[j];
        }
      r1 = rsqrtf(row_sum<RT>(ss, red0, group, tid) * inv_h + a.eps);
      if (a.r1 != nullptr && tid == 0) a.r1[row] = r1;
    }
    float nx[NV][VEC];
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = tid + k * RT;
      if (i < nv) {
        float u[VEC], v[VEC];
        bv[k].get(u);
        if (w1 != nullptr) {
          Vec<T, VEC> wv;
          wv.load(w1 + i * VEC);
          wv.get(v);
#pragma unroll
          for (int j = 0; j < VEC; ++j) u[j] *= r1 * v[j];
        }
        if (gate != nullptr) {
          Vec<T, VEC> gv;
          gv.load(gate + i * VEC);
          gv.get(v);
#pragma unroll
          for (int j = 0; j < VEC; ++j) u[j] *= v[j];
        }
        if constexpr (DROP) {
          drop_factors<VEC>(a.drop, seed, factor, base + static_cast<int64_t>(i) * VEC, v);
#pragma unroll
          for (int j = 0; j < VEC; ++j) u[j] = masked(u[j], v[j]);
        }
        xv[k].get(v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          nx[k][j] = v[j] + a.scale * u[j];
          ss += nx[k][j] * nx[k][j];
        }
        Vec<T, VEC>::store(static_cast<T*>(a.xnew) + base + static_cast<int64_t>(i) * VEC, nx[k]);
      }
    }
    if (w2 != nullptr) {
      // from x' in 32 bits: y carries one rounding, its own
      const float r2 = rsqrtf(row_sum<RT>(ss, red1, group, tid) * inv_h + a.eps);
      if (a.r2 != nullptr && tid == 0) a.r2[row] = r2;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int i = tid + k * RT;
        if (i < nv) {
          Vec<T, VEC> wv;
          float v[VEC];
          wv.load(w2 + i * VEC);
          wv.get(v);
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[j] *= nx[k][j] * r2;
          Vec<T, VEC>::store(static_cast<T*>(a.y) + base + static_cast<int64_t>(i) * VEC, v);
        }
      }
    }
    // without one of the two sums a group's slots are written again after one barrier only
    if (RT > 32 && ((w1 != nullptr) != (w2 != nullptr))) named_bar_sync(1 + group, RT);
  }
}

template <typename T, int VEC, int NV, int RT, bool DROP>
__global__ void __launch_bounds__(RT > 256 ? RT : 256)
    join_bwd_k(const JoinArgs a, float factor) {
  __shared__ float red_all[2][32];
  const int group = threadIdx.x / RT, tid = threadIdx.x % RT, groups = blockDim.x / RT;
  float* red0 = red_all[0] + group * (RT / 32);
  float* red1 = red_all[1] + group * (RT / 32);
  const int nv = a.H / VEC;
  const T* xn = static_cast<const T*>(a.xnew);
  const T* b = static_cast<const T*>(a.b);
  const T* w1 = static_cast<const T*>(a.w1);
  const T* gate = static_cast<const T*>(a.gate);
  const T* w2 = static_cast<const T*>(a.w2);
  const T* dxn = static_cast<const T*>(a.dxnew);
  const T* dy = static_cast<const T*>(a.dy);
  uint64_t seed = 0;
  if constexpr (DROP)
    seed = a.drop.seed_ptr != nullptr ? static_cast<uint64_t>(*a.drop.seed_ptr) : a.drop.seed;
  const float inv_h = 1.f / a.H;
  const bool need_b = w1 != nullptr || a.dgate != nullptr;  // b itself enters the gradients
  const bool branch = a.db != nullptr || a.dgate != nullptr || a.dw1 != nullptr;
  float s1[NV][VEC], s2[NV][VEC];  // columns' sums of t bh and dy xh
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s1[k][j] = s2[k][j] = 0.f;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * groups + group; row < a.T;
       row += static_cast<int64_t>(gridDim.x) * groups) {
    const int64_t base = row * a.H;
    Vec<T, VEC> bv[NV], xv[NV], yv[NV], gv[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = tid + k * RT;
      const int64_t at = base + static_cast<int64_t>(i) * VEC;
      if (i < nv) {
        if (dy != nullptr) {
          yv[k].load_once(dy + at);
          xv[k].load_once(xn + at);
        }
        if (dxn != nullptr) gv[k].load_once(dxn + at);
        if (branch && need_b) bv[k].load_once(b + at);
      }
    }
    float g[NV][VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (dxn != nullptr && tid + k * RT < nv) {
        gv[k].get(g[k]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[k][j] = 0.f;
      }
    }
    if (dy != nullptr) {
      const float r2 = a.r2[row];
      float dot = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int i = tid + k * RT;
        if (i < nv) {
          float d[VEC], v[VEC], w[VEC];
          Vec<T, VEC> wv;
          wv.load(w2 + i * VEC);
          yv[k].get(d);
          xv[k].get(v);
          wv.get(w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float dxh = d[j] * (v[j] * r2);
            s2[k][j] += dxh;
            dot += dxh * w[j];
          }
        }
      }
      const float mean = row_sum<RT>(dot, red0, group, tid) * inv_h;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int i = tid + k * RT;
        if (i < nv) {
          float d[VEC], v[VEC], w[VEC];
          Vec<T, VEC> wv;
          wv.load(w2 + i * VEC);
          yv[k].get(d);
          xv[k].get(v);
          wv.get(w);
#pragma unroll
          for (int j = 0; j < VEC; ++j) g[k][j] += r2 * (d[j] * w[j] - v[j] * r2 * mean);
        }
      }
    }
    if (a.dx != nullptr) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int i = tid + k * RT;
        if (i < nv)
          Vec<T, VEC>::store(static_cast<T*>(a.dx) + base + static_cast<int64_t>(i) * VEC, g[k]);
      }
    }
    if (branch) {
      const float r1 = w1 != nullptr ? a.r1[row] : 1.f;
      float dot = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int i = tid + k * RT;
        if (i < nv) {
          float v[VEC];
          if constexpr (DROP) {
            drop_factors<VEC>(a.drop, seed, factor, base + static_cast<int64_t>(i) * VEC, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) g[k][j] = masked(g[k][j], v[j]);
          }
#pragma unroll
          for (int j = 0; j < VEC; ++j) g[k][j] *= a.scale;
          float bh[VEC];
          if (need_b) {
            bv[k].get(bh);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              bh[j] *= r1;
              s1[k][j] += DROP && v[j] == 0.f ? 0.f : g[k][j] * bh[j];
            }
          }
          if (gate != nullptr) {
            Vec<T, VEC> wv;
            wv.load(gate + i * VEC);
            wv.get(v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) g[k][j] *= v[j];
          }
          if (w1 != nullptr) {
            Vec<T, VEC> wv;
            wv.load(w1 + i * VEC);
            wv.get(v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              g[k][j] *= v[j];
              dot += g[k][j] * bh[j];
            }
          }
        }
      }
      if (w1 != nullptr) {
        const float mean = row_sum<RT>(dot, red1, group, tid) * inv_h;
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if (tid + k * RT < nv) {
            float bh[VEC];
            bv[k].get(bh);
#pragma unroll
            for (int j = 0; j < VEC; ++j) g[k][j] = r1 * (g[k][j] - bh[j] * r1 * mean);
          }
      }
      if (a.db != nullptr) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int i = tid + k * RT;
          if (i < nv)
            Vec<T, VEC>::store(static_cast<T*>(a.db) + base + static_cast<int64_t>(i) * VEC, g[k]);
        }
      }
    }
    if (RT > 32 && ((branch && w1 != nullptr) != (dy != nullptr))) named_bar_sync(1 + group, RT);
  }
  if (a.partials == nullptr) return;
  // the groups of the CTA one after the other, through this CTA's part of the workspace
  float* p = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * a.H;
  for (int q = 0; q < groups; ++q) {
    if (q == group) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int i = tid + k * RT;
        if (i < nv) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float* at = p + i * VEC + j;
            at[0] = (q == 0 ? 0.f : at[0]) + s1[k][j];
            at[a.H] = (q == 0 ? 0.f : at[a.H]) + s2[k][j];
          }
        }
      }
    }
    __syncthreads();
  }
}

// The CTAs' column sums, 32 columns a block, 32 threads a column, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) join_cols_k(const JoinArgs a, int blocks) {
  __shared__ float t1[32][33], t2[32][33];
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
  s1 = warp_sum(t1[tx][ty]);
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

// y = m * x, eight elements (one block of the generator) a thread and turn.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) dropout_k(const T* __restrict__ x, T* __restrict__ y,
                                                 int64_t n, const DropArgs d, float factor) {
  constexpr int VEC = 16 / sizeof(T);
  const uint64_t seed =
      d.seed_ptr != nullptr ? static_cast<uint64_t>(*d.seed_ptr) : d.seed;
  const int64_t blocks = (n + 7) / 8;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < blocks;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t e = i * 8;
    float v[8], m[8];
    if (ALIGNED && e + 8 <= n) {
      Vec<T, VEC> in[8 / VEC];
#pragma unroll
      for (int q = 0; q < 8 / VEC; ++q) in[q].load_once(x + e + q * VEC);
      drop_factors<8>(d, seed, factor, e, m);
#pragma unroll
      for (int q = 0; q < 8 / VEC; ++q) {
        in[q].get(v + q * VEC);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[q * VEC + j] = masked(v[q * VEC + j], m[q * VEC + j]);
        Vec<T, VEC>::store(y + e + q * VEC, v + q * VEC);
      }
    } else {
      drop_factors<8>(d, seed, factor, e, m);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e + j < n) y[e + j] = from_f<T>(masked(to_f<T>(x[e + j]), m[j]));
    }
  }
}

// ---------------------------------------------------------------- host side
int elem_bytes(int type) { return type == kStreamFloat ? 4 : 2; }
bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool join_aligned(const JoinArgs& a) {
  return a.H % (16 / elem_bytes(a.type)) == 0 && al16(a.x) && al16(a.b) && al16(a.w1) &&
         al16(a.gate) && al16(a.w2) && al16(a.xnew) && al16(a.y) && al16(a.dxnew) && al16(a.dy) &&
         al16(a.dx) && al16(a.db);
}

// Calls f with the (VEC, NV, RT) of a row: the fewest threads that hold it in a few vectors.
template <typename T, typename F>
int with_shape(const JoinArgs& a, F f) {
  constexpr int V = 16 / sizeof(T);
  if (join_aligned(a)) {
    const int n = a.H / V;
    if (n <= 32) return f(std::integral_constant<int, V>(), std::integral_constant<int, 1>(),
                          std::integral_constant<int, 32>());
    if (n <= 128) return f(std::integral_constant<int, V>(), std::integral_constant<int, 1>(),
                           std::integral_constant<int, 128>());
    if (n <= 512) return f(std::integral_constant<int, V>(), std::integral_constant<int, 2>(),
                           std::integral_constant<int, 256>());
    if (n <= kJoinMaxVecs)
      return f(std::integral_constant<int, V>(), std::integral_constant<int, 4>(),
               std::integral_constant<int, 512>());
    return -2;
  }
  if (a.H <= 1024) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 4>(),
                            std::integral_constant<int, 256>());
  if (a.H <= kJoinMaxOdd)
    return f(std::integral_constant<int, 1>(), std::integral_constant<int, 16>(),
             std::integral_constant<int, 512>());
  return -2;
}

template <typename F>
int with_type(int type, F f) {
  if (type == kStreamBf16) return f(__nv_bfloat16());
  if (type == kStreamHalf) return f(__half());
  return f(float());
}

// Rows side by side in a CTA: as many as fill 256 threads, fewer where that leaves SMs idle.
int groups_of(int rt, int64_t rows, int num_sms) {
  int g = rt >= 256 ? 1 : 256 / rt;
  while (g > 1 && (rows + g - 1) / g < num_sms) g /= 2;
  return g;
}

// CTAs of a persistent launch: one for each `groups` rows, at most what is resident at once.
template <typename K>
int grid_of(K kern, int threads, int64_t rows, int groups, int num_sms) {
  const int64_t want = rows > 0 ? (rows + groups - 1) / groups : 1;
  if (want <= num_sms) return static_cast<int>(want);
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, 0) != cudaSuccess || n < 1)
    n = 1;
  const int64_t most = static_cast<int64_t>(num_sms) * n;
  return static_cast<int>(want < most ? want : most);
}

}  // namespace

bool join_width_ok(int H, int type) {
  const int v = 16 / elem_bytes(type);
  return H % v == 0 ? H / v <= kJoinMaxVecs : H <= kJoinMaxOdd;
}

int join_fwd(const JoinArgs& a, int num_sms, cudaStream_t s) {
  if (a.T == 0) return 0;
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    return with_shape<T>(a, [&](auto vec, auto nv, auto rt) {
      constexpr int VEC = decltype(vec)::value, NV = decltype(nv)::value, RT = decltype(rt)::value;
      const int groups = groups_of(RT, a.T, num_sms), threads = RT * groups;
      const auto go = [&](auto kern) {
        kern<<<grid_of(kern, threads, a.T, groups, num_sms), threads, 0, s>>>(a, a.drop.factor());
        return static_cast<int>(cudaGetLastError());
      };
      return a.drop.threshold > 0 ? go(join_fwd_k<T, VEC, NV, RT, true>)
                                  : go(join_fwd_k<T, VEC, NV, RT, false>);
    });
  });
}

template <typename F>
static int bwd_shape(const JoinArgs& a, F f) {
  return with_type(a.type, [&](auto t) {
    using T = decltype(t);
    return with_shape<T>(a, [&](auto vec, auto nv, auto rt) {
      constexpr int VEC = decltype(vec)::value, NV = decltype(nv)::value, RT = decltype(rt)::value;
      return a.drop.threshold > 0 ? f(t, join_bwd_k<T, VEC, NV, RT, true>, RT)
                                  : f(t, join_bwd_k<T, VEC, NV, RT, false>, RT);
    });
  });
}

int join_bwd_blocks(const JoinArgs& a, int num_sms) {
  return bwd_shape(a, [&](auto, auto kern, int rt) {
    const int groups = groups_of(rt, a.T, num_sms);
    return grid_of(kern, rt * groups, a.T, groups, num_sms);
  });
}

int join_bwd(const JoinArgs& a, int blocks, int num_sms, cudaStream_t s) {
  return bwd_shape(a, [&](auto t, auto kern, int rt) {
    using T = decltype(t);
    const int groups = groups_of(rt, a.T, num_sms);
    kern<<<blocks, rt * groups, 0, s>>>(a, a.drop.factor());
    if (a.partials != nullptr)
      join_cols_k<T><<<(a.H + 31) / 32, 1024, 0, s>>>(a, blocks);
    return static_cast<int>(cudaGetLastError());
  });
}

int dropout_run(const void* x, void* y, int64_t n, int type, const DropArgs& d, int num_sms,
                cudaStream_t s) {
  if (n == 0) return 0;
  const int64_t want = ((n + 7) / 8 + 255) / 256, most = static_cast<int64_t>(num_sms) * 8;
  const unsigned grid = static_cast<unsigned>(want < most ? want : most);
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    if (al16(x) && al16(y))
      dropout_k<T, true><<<grid, 256, 0, s>>>(static_cast<const T*>(x), static_cast<T*>(y), n, d,
                                              d.factor());
    else
      dropout_k<T, false><<<grid, 256, 0, s>>>(static_cast<const T*>(x), static_cast<T*>(y), n, d,
                                               d.factor());
    return static_cast<int>(cudaGetLastError());
  });
}

}  // namespace cfb
