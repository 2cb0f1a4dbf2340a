// Attention over the 8-bit paged KV cache (sm_100a): decode tokens and short chunks.
//
//   s_j = scale * ks[b(j)] * (q . cK_j),  o = sum_j softmax(s)_j * vs[b(j)] * cV_j
//
// for each row (new token, query head) over the cached tokens j at or before its position.
//
// A step reads every cached byte once and does little else, so the kernel is built to keep
// bytes in flight: codes go from global memory straight into tensor-core fragments, with
// no shared memory, barrier or wait between.  Both products take the cache as the A operand
// of m16n8k16 and the rows of one KV head (tokens x grouped heads) as its 8 columns,
//   S^T[16 tokens, 8 rows] = K[16, D] Q^T      O^T[D, 8 rows] += V^T[D, 16] P^T,
// which wastes nothing on the usual groups of up to eight query heads.  A contraction may
// visit its axis in any order that both operands share, and an output axis may be dealt to
// rows at will; the orders below are chosen so that each lane's share of a page is whole
// 16-byte pieces of it (D = 64: 8-byte pieces of V).  tcgen05 needs 64 rows and operands
// in shared memory: eight times the work and a staging pass for a kernel that waits on HBM.
//
// Codes become f16 exactly; q is scaled by a power of two per row into f16 range, where a
// bf16 q is exact too.  Scores, maxima, sums and the output accumulate in fp32; the
// probabilities are rounded to f16 (11 bits, against 8 of bf16).
// V's block scale cannot be taken out of the sum over blocks, so it goes into the
// exponent: with w_j = s_j + log2 vs[b(j)] and M a running bound of w,
//   P_j = 2^(w_j - M),  O = sum P_j cV_j,  l = sum P_j / vs[b(j)],  o = O / l.
// M moves only when some w exceeds it by more than 2^8 (then by a warp-wide maximum), which
// leaves one vote per page in the usual case.
#include "paged8.cuh"

namespace cfb {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 4;
constexpr float kGrow = 8.f;           // log2 of how far P may exceed 1
constexpr float kTinyScale = 7.888609e-31f;  // 2^-100: V blocks below it count as zeros

struct AttnParams {
  P8Cache c;
  P8Seqs s;
  const void* q;
  int64_t q_stride;
  void* out;
  int64_t N;
  int Hq, G, splits, row_tiles;
  float scale_log2;
  float* ws_o;
  float* ws_lse;
  float* ws_s;
  int64_t s_stride;
  int* err;
};

__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 ld_stream16(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream8(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
               : "=r"(v.x), "=r"(v.y)
               : "l"(p));
  return v;
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

// One lane's share of a page: g = lane / 4, t = lane % 4.
//   k[i][h]: token g + 8 i, bytes [64 h + 16 t, + 16)   -> k-steps 4 h .. 4 h + 3
//   v[i]:    token {2t, 2t+1, 2t+8, 2t+9}[i], bytes [g D / 8, + D / 8)
template <int D>
struct PageFrag {
  static constexpr int KH = D / 64;
  static constexpr int VW = D / 32;  // words of one token's piece
  uint4 k[2][KH];
  uint32_t v[4][VW];
  __device__ __forceinline__ void load(const uint8_t* p, int g, int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < KH; ++h) k[i][h] = ld_stream16(p + (g + 8 * i) * D + 64 * h + 16 * t);
    const uint8_t* pv = p + kP8Page * D + g * (D / 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = 2 * t + (i & 1) + 8 * (i >> 1);
      if constexpr (D == 128) {
        const uint4 x = ld_stream16(pv + tok * D);
        v[i][0] = x.x;
        v[i][1] = x.y;
        v[i][2] = x.z;
        v[i][3] = x.w;
      } else {
        const uint2 x = ld_stream8(pv + tok * D);
        v[i][0] = x.x;
        v[i][1] = x.y;
      }
    }
  }
};

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// NB: 8-row column tiles of a CTA (8 * NB rows of one KV head).
template <typename T, int FMT, int D, int NB, bool MASS>
__global__ void __launch_bounds__(kWarps * 32) p8_attn_kernel(const AttnParams p) {
  constexpr int R = 8 * NB;
  constexpr int KH = D / 64, KS = D / 16, MT = D / 16;
  constexpr int DL = D / 8;  // output dims of a lane
  __shared__ float s_m[kWarps][R], s_l[kWarps][R];
  __shared__ __align__(16) float s_o[kWarps][R][D];

  const int split = blockIdx.x % p.splits, rt = blockIdx.x / p.splits;
  const int h = blockIdx.y, seq = blockIdx.z;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane >> 2, t = lane & 3;
  const int row0 = __ldg(p.s.cu_q + seq);
  const int q_len = __ldg(p.s.cu_q + seq + 1) - row0;
  if (row0 < 0 || q_len < 0 || static_cast<int64_t>(row0) + q_len > p.N) {
    if (threadIdx.x == 0) report_error(p.err, kErrBounds, 70);
    return;
  }
  const int rows = q_len * p.G;       // rows of this KV head
  const int first_row = rt * R;
  if (rt == p.row_tiles - 1 && rows > first_row + R && threadIdx.x == 0)
    report_error(p.err, kErrBounds, 71);  // a chunk longer than max_q_len
  if (first_row >= rows) return;
  const int kv = p8_len(p.s.kv_lens, seq, p.s.max_pages, p.err, 72);
  // row r is token r / G and head r % G; its visible keys are [0, start + token + 1)
  const int start = kv - q_len;
  const int last_tok = (min(rows, first_row + R) - 1) / p.G;
  const int n_keys = max(0, start + last_tok + 1);
  const int n_pages = (n_keys + kP8Page - 1) / kP8Page;
  // even ranges of this row tile's own pages, at least two pages a warp
  const int per = max(2 * kWarps, (n_pages + p.splits - 1) / p.splits);
  const int p_begin = split * per, p_end = min(n_pages, p_begin + per);
  auto out_row = [&](int r) {  // row of out / ws (token-major, Hq heads)
    return static_cast<int64_t>(row0 + r / p.G) * p.Hq + h * p.G + r % p.G;
  };
  if (p_begin >= p_end && split > 0) {
    for (int r = threadIdx.x; r < R; r += blockDim.x)
      if (first_row + r < rows) p.ws_lse[out_row(first_row + r) * p.splits + split] = -INFINITY;
    return;
  }
  const int32_t* table = p.s.table + static_cast<int64_t>(seq) * p.s.max_pages;
  const int first = p_begin + warp;
  const int count = first < p_end ? (p_end - first + kWarps - 1) / kWarps : 0;

  // Pages of this warp, 32 at a time: lane i looks up the i-th (pool offset, scales).
  int64_t ids = 0, ids_next = 0;
  float2 sc = make_float2(0.f, 0.f), sc_next = sc;
  auto lookup = [&](int j) -> int64_t {
    return j < count ? p8_page(table, first + kWarps * j, p.c.num_pages, p.err, 73) * p.c.Hkv + h
                     : 0;
  };
  auto scales_of = [&](int j, int64_t ph) {
    return j < count ? __ldg(reinterpret_cast<const float2*>(p.c.scales) + ph)
                     : make_float2(0.f, 0.f);
  };
  ids = lookup(lane);
  sc = scales_of(lane, ids);
  if (count > 32) {
    ids_next = lookup(32 + lane);
    sc_next = scales_of(32 + lane, ids_next);
  }
  PageFrag<D> cur, nxt;
  if (count > 0) cur.load(p.c.codes + __shfl_sync(kFull, ids, 0) * (2 * kP8Page * D), g, t);

  // q as B fragments in f16, scaled by a power of two per row
  uint32_t qb[NB][KS][2];
  float qs[NB][2];   // of rows 2 t, 2 t + 1: scale * log2(e) * the power of two undone
  int lim[NB][2];    // their visible keys
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = first_row + nb * 8 + g;
    const bool live = r < rows;
    const T* qr = static_cast<const T*>(p.q) +
                  static_cast<int64_t>(row0 + (live ? r / p.G : 0)) * p.q_stride +
                  (h * p.G + (live ? r % p.G : 0)) * D;
    float f[KS][4];
    uint32_t top = 0;
#pragma unroll
    for (int hh = 0; hh < KH; ++hh)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (live) u = __ldg(reinterpret_cast<const uint4*>(qr + 64 * hh + 16 * t) + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = P8Io<T>::unpack(word_of(u, e));
          float* d = &f[hh * 4 + c * 2 + (e >> 1)][(e & 1) * 2];
          d[0] = x.x;
          d[1] = x.y;
          top = max(top,
                    max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu));
        }
      }
    top = max(top, __shfl_xor_sync(kFull, top, 1));
    top = max(top, __shfl_xor_sync(kFull, top, 2));
    // 2^-e with 2^e the largest power of two in the row's magnitude
    const int ex = min(max(static_cast<int>(top >> 23), 27), 227);
    const float down = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
    const float up = __uint_as_float(static_cast<uint32_t>(ex) << 23) * p.scale_log2;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      qb[nb][k][0] = half2_of(f[k][0] * down, f[k][1] * down);
      qb[nb][k][1] = half2_of(f[k][2] * down, f[k][3] * down);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      qs[nb][i] = __shfl_sync(kFull, up, (2 * t + i) * 4);
      const int rr = first_row + nb * 8 + 2 * t + i;
      lim[nb][i] = rr < rows ? start + rr / p.G + 1 : 0;
    }
  }

  float o[NB][MT][4];
  float M[NB][2], l[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int j = 0; j < MT; ++j) o[nb][j][0] = o[nb][j][1] = o[nb][j][2] = o[nb][j][3] = 0.f;
    M[nb][0] = M[nb][1] = -INFINITY;
    l[nb][0] = l[nb][1] = 0.f;
  }
  const int min_lim = start + first_row / p.G + 1;  // every row of the tile sees these keys
  float lv_last = 0.f, rv_last = 1.f;

  auto page_step = [&](PageFrag<D>& f, int j) {
    const float ks = __shfl_sync(kFull, sc.x, j & 31), vs = __shfl_sync(kFull, sc.y, j & 31);
    const int key0 = (first + kWarps * j) * kP8Page;
    // ---- S^T = K Q^T
    float s[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
#pragma unroll
    for (int hh = 0; hh < KH; ++hh)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t a0, a1, a2, a3;
        p8_to_half<FMT>(word_of(f.k[0][hh], w), a0, a2);
        p8_to_half<FMT>(word_of(f.k[1][hh], w), a1, a3);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          mma_f16(s[nb], a0, a1, a2, a3, qb[nb][hh * 4 + w][0], qb[nb][hh * 4 + w][1]);
      }
    // ---- w = s + log2(vs); a V block of (nearly) zeros adds to l alone
    const bool has_v = !(vs < kTinyScale);
    const bool fine = vs <= 3.402823466e38f;
    if (has_v && fine) {
      lv_last = __log2f(vs);
      rv_last = __fdividef(1.f, vs);
    }
    const float lv = fine ? lv_last : vs - vs, rv = rv_last;  // not finite: NaN
    const bool edge = key0 + kP8Page > min_lim;
    bool grow = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = e & 1;  // row 2 t + i, token g + 8 (e / 2)
        float x = s[nb][e] * (ks * qs[nb][i]);
        const bool hidden = edge && key0 + g + 8 * (e >> 1) >= lim[nb][i];
        if constexpr (MASS) {
          const int r = first_row + nb * 8 + 2 * t + i;
          if (r < rows)
            p.ws_s[out_row(r) * p.s_stride + key0 + g + 8 * (e >> 1)] = x;
        }
        s[nb][e] = hidden ? -INFINITY : x + lv;
        grow |= s[nb][e] > M[nb][i] + kGrow;
      }
    }
    if (__any_sync(kFull, grow)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float m = fmaxf(s[nb][i], s[nb][2 + i]);
          m = fmaxf(m, __shfl_xor_sync(kFull, m, 4));
          m = fmaxf(m, __shfl_xor_sync(kFull, m, 8));
          m = fmaxf(m, __shfl_xor_sync(kFull, m, 16));
          m = fmaxf(m, M[nb][i]);
          const float a = M[nb][i] == -INFINITY ? 0.f : ex2f(M[nb][i] - m);
          M[nb][i] = m;
          l[nb][i] *= a;
#pragma unroll
          for (int jj = 0; jj < MT; ++jj) {
            o[nb][jj][i] *= a;
            o[nb][jj][2 + i] *= a;
          }
        }
    }
    uint32_t pb[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float e4[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float base = M[nb][i] == -INFINITY ? 0.f : M[nb][i];  // nothing visible yet
        e4[i] = ex2f(s[nb][i] - base);
        e4[2 + i] = ex2f(s[nb][2 + i] - base);
        const float sum = e4[i] + e4[2 + i];
        l[nb][i] += sum == 0.f ? 0.f : sum * rv;
      }
      pb[nb][0] = has_v ? transpose8x8(half2_of(e4[0], e4[1])) : 0u;
      pb[nb][1] = has_v ? transpose8x8(half2_of(e4[2], e4[3])) : 0u;
    }
    // ---- O^T += V^T P^T; codes past the last visible key are never looked at
    const int live = n_keys - key0;
    if (live < kP8Page) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (2 * t + (i & 1) + 8 * (i >> 1) >= live)
#pragma unroll
          for (int w = 0; w < PageFrag<D>::VW; ++w) f.v[i][w] = 0u;
    }
#pragma unroll
    for (int w = 0; w < PageFrag<D>::VW; ++w) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {  // bytes 4 w + 2 hf, + 1 of the piece
        const uint32_t sel = hf == 0 ? 0x5140 : 0x7362;
        uint32_t a0, a1, a2, a3;
        p8_to_half<FMT>(__byte_perm(f.v[0][w], f.v[1][w], sel), a0, a1);
        p8_to_half<FMT>(__byte_perm(f.v[2][w], f.v[3][w], sel), a2, a3);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          mma_f16(o[nb][2 * w + hf], a0, a1, a2, a3, pb[nb][0], pb[nb][1]);
      }
    }
  };
  auto fetch = [&](PageFrag<D>& f, int j) {  // page j's codes; j in the current or next 32
    const int64_t ph = __shfl_sync(kFull, (j & ~31) == 0 || (j & 31) ? ids : ids_next, j & 31);
    f.load(p.c.codes + ph * (2 * kP8Page * D), g, t);
  };
  for (int j = 0; j < count; j += 2) {
    if (j + 1 < count) fetch(nxt, j + 1);
    page_step(cur, j);
    if (j + 1 < count) {
      if (j + 2 < count) fetch(cur, j + 2);
      page_step(nxt, j + 1);
    }
    if (((j + 2) & 31) == 0) {  // the next 32 pages become current
      ids = ids_next;
      sc = sc_next;
      ids_next = lookup(j + 2 + 32 + lane);
      sc_next = scales_of(j + 2 + 32 + lane, ids_next);
    }
  }

  // ---- join the warps
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x = l[nb][i];
      x += __shfl_xor_sync(kFull, x, 4);
      x += __shfl_xor_sync(kFull, x, 8);
      x += __shfl_xor_sync(kFull, x, 16);
      const int r = nb * 8 + 2 * t + i;
      if (g == 0) {
        s_m[warp][r] = M[nb][i];
        s_l[warp][r] = x;
      }
      // dims g D / 8 + 2 j (+ 1): element j of the lane's piece, two per m-tile
#pragma unroll
      for (int j = 0; j < MT; j += 2)
        *reinterpret_cast<float4*>(&s_o[warp][r][g * DL + 2 * j]) =
            make_float4(o[nb][j][i], o[nb][j][2 + i], o[nb][j + 1][i], o[nb][j + 1][2 + i]);
    }
  __syncthreads();
  for (int e = threadIdx.x; e < R * (D / 4); e += blockDim.x) {
    const int r = e / (D / 4), d = (e % (D / 4)) * 4;
    if (first_row + r >= rows) continue;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_m[w][r]);
    float den = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (s_m[w][r] == -INFINITY && s_l[w][r] == 0.f) continue;
      const float x = ex2f(s_m[w][r] - m);
      const float4 y = *reinterpret_cast<const float4*>(&s_o[w][r][d]);
      den += s_l[w][r] * x;
      acc.x += y.x * x;
      acc.y += y.y * x;
      acc.z += y.z * x;
      acc.w += y.w * x;
    }
    const float inv = den == 0.f ? 0.f : __fdiv_rn(1.f, den);  // no visible key: 0
    acc.x *= inv;
    acc.y *= inv;
    acc.z *= inv;
    acc.w *= inv;
    const int64_t orow = out_row(first_row + r);
    if (p.splits == 1) {
      uint2 u;
      u.x = P8Io<T>::pack(acc.x, acc.y);
      u.y = P8Io<T>::pack(acc.z, acc.w);
      *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + orow * D + d) = u;
    } else {
      *reinterpret_cast<float4*>(p.ws_o + (orow * p.splits + split) * D + d) = acc;
    }
    if (d == 0 && p.ws_lse != nullptr)
      p.ws_lse[orow * p.splits + split] = den == 0.f ? -INFINITY : m + log2f(den);
  }
}

// Joins the splits of a row: out = sum 2^(lse_s - L) o_s with L = log2 sum 2^lse_s, and
// leaves L in the row's first lse slot for the weights.
template <typename T>
__global__ void __launch_bounds__(128)
    p8_combine_kernel(const float* __restrict__ ws_o, float* __restrict__ ws_lse,
                      T* __restrict__ out, int64_t rows, int splits, int D) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (row >= rows) return;
  float* lse = ws_lse + row * splits;
  float m = -INFINITY;
  for (int s = lane; s < splits; s += 32) m = fmaxf(m, lse[s]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
  const float base = m == -INFINITY ? 0.f : m;
  float den = 0.f;
  for (int s = 0; s < splits; ++s) den += ex2f(lse[s] - base);
  const float inv = den == 0.f ? 0.f : __fdiv_rn(1.f, den);
  for (int d = lane * 2; d < D; d += 64) {
    float2 acc = make_float2(0.f, 0.f);
    for (int s = 0; s < splits; ++s) {
      const float w = ex2f(lse[s] - base);
      if (w == 0.f) continue;
      const float2 x = *reinterpret_cast<const float2*>(ws_o + (row * splits + s) * D + d);
      acc.x += w * x.x;
      acc.y += w * x.y;
    }
    *reinterpret_cast<uint32_t*>(out + row * D + d) = P8Io<T>::pack(acc.x * inv, acc.y * inv);
  }
  __syncwarp();
  if (lane == 0) lse[0] = den == 0.f ? -INFINITY : base + log2f(den);
}

// mass_out[j] = mass_in[j] + sum over the KV head's rows of 2^(s_j - L), in row order.
__global__ void __launch_bounds__(128)
    p8_mass_kernel(P8Cache c, P8Seqs s, const float* __restrict__ ws_s, int64_t s_stride,
                   const float* __restrict__ lse, int splits, int Hq, int G,
                   const float* __restrict__ mass_in, float* __restrict__ mass_out, int* err) {
  const int seq = blockIdx.z, h = blockIdx.y;
  const int kv = p8_len(s.kv_lens, seq, s.max_pages, err, 74);
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= kv) return;
  const int row0 = __ldg(s.cu_q + seq), q_len = __ldg(s.cu_q + seq + 1) - row0;
  const int start = kv - q_len;
  const int64_t page = p8_page(s.table + static_cast<int64_t>(seq) * s.max_pages, j / kP8Page,
                               c.num_pages, err, 75);
  float w = 0.f;
  for (int tok = max(0, j - start); tok < q_len; ++tok)
    for (int g = 0; g < G; ++g) {
      const int64_t row = static_cast<int64_t>(row0 + tok) * Hq + h * G + g;
      w += ex2f(ws_s[row * s_stride + j] - lse[row * splits]);
    }
  const int64_t at = (page * c.Hkv + h) * kP8Page + j % kP8Page;
  mass_out[at] = mass_in[at] + w;
}

template <typename T, int FMT, int D, bool MASS>
int launch_nb(const AttnParams& p, int rows, cudaStream_t st) {
  AttnParams a = p;
  const int nb = rows <= 8 ? 1 : 2;
  a.row_tiles = (rows + 8 * nb - 1) / (8 * nb);
  const int64_t gx = static_cast<int64_t>(a.splits) * a.row_tiles;
  if (gx > 0x7fffffff) return -3;
  const dim3 grid(static_cast<unsigned>(gx), a.c.Hkv, a.s.num_seqs);
  if (nb == 1)
    p8_attn_kernel<T, FMT, D, 1, MASS><<<grid, kWarps * 32, 0, st>>>(a);
  else
    p8_attn_kernel<T, FMT, D, 2, MASS><<<grid, kWarps * 32, 0, st>>>(a);
  return 0;
}

template <typename T, int FMT, int D>
int launch_attn(const AttnParams& p, const P8Attn& a, int rows, cudaStream_t st) {
  const bool mass = a.mass_out != nullptr;
  const int rc = mass ? launch_nb<T, FMT, D, true>(p, rows, st)
                      : launch_nb<T, FMT, D, false>(p, rows, st);
  if (rc) return rc;
  if (p.splits > 1) {
    const int rc = p8_combine(a, D, st);
    if (rc) return rc;
  }
  if (mass) {
    const int L = p.s.max_pages * kP8Page;
    p8_mass_kernel<<<dim3((L + 127) / 128, p.c.Hkv, p.s.num_seqs), 128, 0, st>>>(
        p.c, p.s, a.ws_s, p.s_stride, a.ws_lse, p.splits, a.Hq, p.G, a.mass_in, a.mass_out,
        p.err);
  }
  return 0;
}

}  // namespace

int p8_combine(const P8Attn& a, int D, cudaStream_t st) {
  const int64_t n = a.N * a.Hq;
  const int64_t grid = (n + 3) / 4;
  if (grid > 0x7fffffff) return -3;
  if (a.type == kP8Bf16)
    p8_combine_kernel<__nv_bfloat16><<<static_cast<unsigned>(grid), 128, 0, st>>>(
        a.ws_o, a.ws_lse, static_cast<__nv_bfloat16*>(a.out), n, a.splits, D);
  else
    p8_combine_kernel<__half><<<static_cast<unsigned>(grid), 128, 0, st>>>(
        a.ws_o, a.ws_lse, static_cast<__half*>(a.out), n, a.splits, D);
  return 0;
}

int p8_attn_splits(const P8Seqs& s, int Hkv, int group, int max_q_len, int num_sms) {
  const int rows = max_q_len * group;
  const int per_tile = rows <= 8 ? 8 : 16;
  const int64_t ctas = static_cast<int64_t>((rows + per_tile - 1) / per_tile) * Hkv * s.num_seqs;
  // about six CTAs for each SM, and at least two pages for each warp
  int64_t sp = (6 * static_cast<int64_t>(num_sms) + ctas - 1) / ctas;
  const int64_t most = (s.max_pages + 2 * kWarps - 1) / (2 * kWarps);
  if (sp > most) sp = most;
  return static_cast<int>(sp < 1 ? 1 : sp);
}

int p8_attention(const P8Cache& c, const P8Seqs& s, const P8Attn& a, int* err,
                 cudaStream_t stream) {
  if (a.N <= 0 || s.num_seqs <= 0) return 0;
  if (s.num_seqs > 65535 || c.Hkv > 65535) return -3;
  AttnParams p;
  p.c = c;
  p.s = s;
  p.q = a.q;
  p.q_stride = a.q_stride;
  p.out = a.out;
  p.N = a.N;
  p.Hq = a.Hq;
  p.G = a.Hq / c.Hkv;
  p.splits = a.splits;
  p.row_tiles = 1;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.ws_o = a.ws_o;
  p.ws_lse = a.ws_lse;
  p.ws_s = a.ws_s;
  p.s_stride = static_cast<int64_t>(s.max_pages) * kP8Page;
  p.err = err;
  const int rows = a.max_q_len * p.G;
  int rc = 0;
  switch (a.type * 4 + c.fmt * 2 + (c.D == 128)) {
    case 0: rc = launch_attn<__nv_bfloat16, kP8Int8, 64>(p, a, rows, stream); break;
    case 1: rc = launch_attn<__nv_bfloat16, kP8Int8, 128>(p, a, rows, stream); break;
    case 2: rc = launch_attn<__nv_bfloat16, kP8E4m3, 64>(p, a, rows, stream); break;
    case 3: rc = launch_attn<__nv_bfloat16, kP8E4m3, 128>(p, a, rows, stream); break;
    case 4: rc = launch_attn<__half, kP8Int8, 64>(p, a, rows, stream); break;
    case 5: rc = launch_attn<__half, kP8Int8, 128>(p, a, rows, stream); break;
    case 6: rc = launch_attn<__half, kP8E4m3, 64>(p, a, rows, stream); break;
    case 7: rc = launch_attn<__half, kP8E4m3, 128>(p, a, rows, stream); break;
    default: return -2;
  }
  return rc ? rc : static_cast<int>(cudaGetLastError());
}

}  // namespace cfb
