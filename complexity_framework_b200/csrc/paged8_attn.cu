// Attention over the 8-bit paged KV cache (sm_100a): decode tokens and short chunks.
//
//   s_j = scale * ks[b(j)] * (q . cK_j),  o = sum_j softmax(s)_j * vs[b(j)] * cV_j
//
// for each row (new token, query head) over the cached tokens j at or before its position.
//
// A step reads every cached byte once and does little else, so the kernel is built to keep
// bytes in flight and instructions few.  Each warp streams pages of one KV head (32 * D
// contiguous bytes) through its own ring in shared memory (cp.async, no barrier); both
// products take the cache as the A operand of m16n8k16 and the rows of the KV head (tokens x
// grouped heads) as its 8 columns,
//   S^T[16 tokens, 8 rows] = K[16, D] Q^T      O^T[D, 8 rows] += V^T[D, 16] P^T,
// which wastes nothing on the usual groups of up to eight query heads.  tcgen05 needs 64 rows
// and 16-bit operands in shared memory: eight times the work and a conversion pass for a
// kernel that waits on HBM.  A contraction may visit its axis in any order that both operands
// share, and an output axis may be dealt to rows at will: the orders are chosen so that a
// lane's share of a page is whole 16-byte pieces (D = 64: 8-byte pieces of V), and the ring is
// swizzled so that a quarter warp's pieces lie in distinct banks.
//
// Codes become f16 exactly: an e4m3 number is an f16 number; an int8 code c becomes the f16
// subnormal (c + 128) 2^-24, which is its byte with the sign bit flipped and needs one byte
// permutation for two codes.  The offset comes out again exactly where it went in: 128 sum(q)
// is subtracted from the score, 128 sum(P) (an MMA against ones, so of the rounded P) from the
// output; the score's 32-bit sum carries 128 sum|q| in place of sum|q c| on the way.
// q is scaled by a power of two per row into f16 range.  A bf16 element is exact there down to
// 2^-17 of the row's largest; below it loses at most 2^-25 of the largest.  (The long chunks'
// products take a bf16 q as it is.)
// Scores, maxima, sums and the output accumulate in fp32; the probabilities are rounded to
// f16 (11 bits, against 8 of bf16).
// V's block scale cannot be taken out of the sum over blocks, so it goes into the exponent:
// with w_j = s_j + log2 vs[b(j)] and M a running bound of w,
//   P_j = 2^(w_j - M),  O = sum P_j cV_j,  l = sum P_j / vs[b(j)],  o = O / l.
// What P loses to f16's subnormals, where a block's vs lies 2^14 or more below the largest
// product's, is at most 2^-25 of that product.
// M moves only when some w exceeds it by more than 2^8 (then by a warp-wide maximum), which
// leaves one vote per page in the usual case.
//
// One CTA takes `chunk` pages of one item (sequence, KV head, row tile); the host picks the
// chunk for a few waves of CTAs from the page table's width, and CTAs past a sequence's own
// length leave at once.  The hardware deals CTAs to SMs as they free up: SMs run up to 18%
// apart on equal work, so equal static shares (57 us for 64 ragged requests, 40 in the next
// version with chunks) wait for the slowest one.  Items of more than one chunk leave normalised
// partial outputs, which p8_finish_kernel joins; a cluster for each item that joins over distributed shared memory was
// slower (39.0 us against 36.3, with weights 60.8 against 49.7, at the time): it needs all its
// CTAs' slots at once.
//
// Measured (D 128, int8, GQA 32/8, whole calls): 64 requests of 129 to 2304 tokens 34.1 us, 4.3
// TB/s, bound by start, last wave and join; 256 of 1000 tokens 86.2 us, 6.1 TB/s (0.95 of a copy).
// 311 warp instructions for a page of one head, 42% of the issue slots.
#include <algorithm>

#include "paged8.cuh"

namespace cfb {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 4;
constexpr int kStages = 4;                   // pages of a warp's ring: two used, two in flight
constexpr int kWholePages = 32;              // up to here an item is one CTA's
constexpr int kMinPages = 32, kMaxPages = 64;  // chunk of a CTA otherwise
constexpr float kGrow = 8.f;                 // log2 of how far P may exceed 1
constexpr float kNone = -1e30f;              // M before any visible key
constexpr float kTinyScale = 7.888609e-31f;  // 2^-100: V blocks below it count as zeros
constexpr float kTwo24 = 16777216.f;

struct AttnParams {
  P8Cache c;
  P8Seqs s;
  const void* q;
  int64_t q_stride;
  void* out;
  int64_t N;
  int Hq, G;
  int row_tiles;               // of the longest chunk of new tokens
  int max_rows;                // its rows: the workspace has no room for more
  int chunk, splits;           // pages of a CTA, CTAs of the longest item
  float scale_log2;
  float* ws_o;                 // [items, splits, R, D] partial outputs (splits > 1)
  float* ws_lse;               // [items, splits, R] (splits > 1 or mass)
  float* ws_s;                 // [items, max_pages * 16, RS] scores (mass)
  int RS;                      // rows of a token's scores: 4 where those are enough, else R
  const float* mass_in;
  float* mass_out;
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
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
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
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Four codes as two f16x2 A-operand registers, (byte 0, byte 1) and (byte 2, byte 3):
// e4m3 as its value; int8 (sign bit flipped by the caller) as (c + 128) 2^-24.
template <int FMT>
__device__ __forceinline__ void operand(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == kP8Int8) {
    lo = __byte_perm(w, 0u, 0x4140);
    hi = __byte_perm(w, 0u, 0x4342);
  } else {
    p8_to_half<FMT>(w, lo, hi);
  }
}
template <int FMT>
__device__ __forceinline__ uint32_t flip(uint32_t w) {
  return FMT == kP8Int8 ? w ^ 0x80808080u : w;
}

template <int D, int NB>
struct AttnCfg {
  static constexpr int R = 8 * NB;
  static constexpr int PAGE_BYTES = 2 * kP8Page * D;
  static constexpr int RING = kWarps * kStages * PAGE_BYTES;
  static constexpr int JOIN = kWarps * R * D * 4;              // reuses the ring
  static constexpr int QF = RING > JOIN ? RING : JOIN;         // q fragments
  static constexpr int ROWS = QF + NB * D * 16;                // per-row values
  static constexpr int SMEM = ROWS + (2 + 2 * kWarps) * R * 4;
  static constexpr int MIN_CTAS = NB <= 2 ? 3 : 2;
  static_assert(SMEM * MIN_CTAS <= 224 * 1024, "shared memory");
};

struct SeqInfo {
  int row0, q_len, kv, rows;  // rows of a KV head: tokens x G
};

__device__ __forceinline__ SeqInfo seq_info(const AttnParams& p, int seq) {
  SeqInfo i;
  i.row0 = __ldg(p.s.cu_q + seq);
  i.q_len = __ldg(p.s.cu_q + seq + 1) - i.row0;
  i.kv = p8_len(p.s.kv_lens, seq, p.s.max_pages, p.err, 72);
  if (i.row0 < 0 || i.q_len < 0 || static_cast<int64_t>(i.row0) + i.q_len > p.N) {
    report_error(p.err, kErrBounds, 70);
    i.q_len = 0;
  }
  if (static_cast<int64_t>(i.q_len) * p.G > p.max_rows) {  // longer than max_q_len
    report_error(p.err, kErrBounds, 71);
    i.rows = p.max_rows;
  } else {
    i.rows = i.q_len * p.G;
  }
  return i;
}

// Where a token's mass is kept.
__device__ __forceinline__ int64_t mass_at(const AttnParams& p, const int32_t* table, int h,
                                           int j) {
  const int64_t pg = p8_page(table, j / kP8Page, p.c.num_pages, p.err, 75);
  return (pg * p.c.Hkv + h) * kP8Page + j % kP8Page;
}
// The weight a token receives: sum over rows of 2^(s_j - lse), in row order.  s: the token's
// scores of the head's first row tile, the next tile's `tile` floats on; r0: the first row that
// sees the token.
template <int R>
__device__ __forceinline__ float weight_of(const float* s, int64_t tile, int r0, int rows,
                                           const float* lse) {
  float w = 0.f;
  for (int b = 0; b < rows; b += R, s += tile)
#pragma unroll 2
    for (int r = 0; r < min(R, rows - b); r += 4) {
      const float4 x = *reinterpret_cast<const float4*>(s + r);
      const int at = b + r;
      if (at >= r0) w += ex2f(x.x - lse[at]);
      if (at + 1 >= r0 && at + 1 < rows) w += ex2f(x.y - lse[at + 1]);
      if (at + 2 >= r0 && at + 2 < rows) w += ex2f(x.z - lse[at + 2]);
      if (at + 3 >= r0 && at + 3 < rows) w += ex2f(x.w - lse[at + 3]);
    }
  return w;
}

// NB: 8-row column tiles of a CTA (R = 8 * NB rows of one KV head).
template <typename T, int FMT, int D, int NB, bool MASS>
__global__ void __launch_bounds__(kWarps * 32, (AttnCfg<D, NB>::MIN_CTAS))
    p8_attn_kernel(const AttnParams p) {
  using Cfg = AttnCfg<D, NB>;
  constexpr int R = Cfg::R;
  constexpr int KH = D / 64, KS = D / 16, MT = D / 16;
  constexpr int DL = D / 8;              // output dims of a lane
  constexpr int VW = D / 32;             // words of a lane's piece of one token's V
  constexpr int PB = Cfg::PAGE_BYTES;
  constexpr int HALF = kP8Page / 2 * D;  // bytes of eight tokens
  constexpr bool kInt8 = FMT == kP8Int8;
  constexpr int U = NB <= 3 ? 2 : 1;     // pages of an iteration: two hide each other's latency
  constexpr int AHEAD = kStages / U - 1; // groups of pages in flight beyond the current one
  extern __shared__ __align__(128) uint8_t smem[];
  float* s_o = reinterpret_cast<float*>(smem);                        // [kWarps][R][D]
  float* s_qs = reinterpret_cast<float*>(smem + Cfg::ROWS);           // [R]
  float* s_qb = s_qs + R;                                             // [R]
  float* s_m = s_qb + R;                                              // [kWarps][R]
  float* s_l = s_m + kWarps * R;                                      // [kWarps][R]
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * (kStages * PB);
  const uint32_t qf = smem_u32(smem + Cfg::QF);
  p8_grid_wait();

  const int split = blockIdx.x % p.splits, rt = blockIdx.x / p.splits;
  const int h = blockIdx.y, seq = blockIdx.z;
  // a page-table entry for each lane, read together with the lengths that say whether it counts
  const int32_t* table = p.s.table + static_cast<int64_t>(seq) * p.s.max_pages;
  const int page = split * p.chunk, first = page + warp;
  const int entry = first + kWarps * lane;
  int id = entry < p.s.max_pages ? __ldg(table + entry) : 0;
  const SeqInfo si = seq_info(p, seq);
  const int rows = si.rows, first_row = rt * R;
  // row r is token r / G and head r % G; it sees the keys [0, start + token + 1)
  const int start = si.kv - si.q_len;
  const int64_t Lp = static_cast<int64_t>(p.s.max_pages) * kP8Page;
  const int64_t item = (static_cast<int64_t>(seq) * p.c.Hkv + h) * p.row_tiles + rt;
  if (first_row >= rows) {
    if (MASS && p.splits == 1 && p.row_tiles == 1)  // cached tokens, none of them new
      for (int j = threadIdx.x; j < si.kv; j += kWarps * 32) {
        const int64_t at = mass_at(p, table, h, j);
        p.mass_out[at] = p.mass_in[at];
      }
    return;
  }
  const int last_tok = (min(rows, first_row + R) - 1) / p.G;
  const int n_keys = max(0, start + last_tok + 1);
  const int min_lim = start + first_row / p.G + 1;  // every row of the tile sees these keys
  const int n_pages = (n_keys + kP8Page - 1) / kP8Page;
  if (page >= n_pages && split > 0) return;
  const int p_end = min(n_pages, page + p.chunk);
  const bool uncut = n_pages <= p.chunk;
  const int count = first < p_end ? (p_end - first + kWarps - 1) / kWarps : 0;

  // constant lane offsets in a page of the ring (see the bank comment above)
  uint32_t cp_off[2], k_off[2], v_off[2];
  {
    const int l8 = lane >> 3, c8 = lane & 7;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int sw = D == 128 ? i * 4 + l8 : (2 * l8) & 7;
      cp_off[i] = l8 * 128 + ((c8 ^ sw) * 16);
      if (D == 128) {
        k_off[i] = g * 128 + (((2 * t + i) ^ g) * 16);
        const int r = 2 * t + i;
        v_off[i] = kP8Page * D + r * 128 + ((g ^ r) * 16);
      } else {
        k_off[i] = (g >> 1) * 128 + ((((g & 1) * 4 + t) ^ ((2 * (g >> 1)) & 7)) * 16);
        v_off[i] = kP8Page * D + t * 128 + (((i * 4 + (g >> 1)) ^ (2 * t)) * 16) + (g & 1) * 8;
      }
    }
  }

  // Pages of this warp (at most 32): lane i holds the i-th one's place and scales (K's; log2
  // and reciprocal of V's, the reciprocal negative for a block of zeros).
  float ks_i = 0.f, lv_i = 0.f, rv_i = 1.f;
  if (lane < count) {
    id = static_cast<int>(p8_checked(id, p.c.num_pages, p.err, 73));
    id = id * p.c.Hkv + h;
    const float2 sc = __ldg(reinterpret_cast<const float2*>(p.c.scales) + id);
    const bool tiny = sc.y < kTinyScale, fine = sc.y <= 3.402823466e38f;
    ks_i = sc.x;
    lv_i = tiny ? -24.f : fine ? __log2f(sc.y) : sc.y - sc.y;  // not finite: NaN
    rv_i = tiny ? -kTwo24 : fine ? __fdividef(1.f, sc.y) : 1.f;
  }
  auto issue = [&](int q) {  // pages U q, ..
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = U * q + u;
      if (j < count) {
        const uint8_t* src =
            p.c.codes + static_cast<int64_t>(__shfl_sync(kFull, id, j)) * PB + lane * 16;
        const uint32_t dst = ring + (j % kStages) * PB;
#pragma unroll
        for (int i = 0; i < PB / 512; ++i) cp_async16(dst + cp_off[i & 1] + i * 512, src + i * 512);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int q = 0; q < AHEAD; ++q) issue(q);

  // ---- q: warp nb turns its eight rows into f16 B fragments in shared memory
  if (warp < NB) {
    const int r = first_row + warp * 8 + g;
    const bool live = r < rows;
    const T* qr = static_cast<const T*>(p.q) +
                  static_cast<int64_t>(si.row0 + (live ? r / p.G : 0)) * p.q_stride +
                  (h * p.G + (live ? r % p.G : 0)) * D + t * (D / 4);
    uint4 u[D / 32];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      u[i] = live ? __ldg(reinterpret_cast<const uint4*>(qr) + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = P8Io<T>::unpack(word_of(u[i], e));
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
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = P8Io<T>::unpack(word_of(u[i], e));
        w[e] = half2_of(x.x * down, x.y * down);
        const float2 y = __half22float2(*reinterpret_cast<__half2*>(&w[e]));
        sum += y.x + y.y;
      }
      *reinterpret_cast<uint4*>(smem + Cfg::QF + ((i * NB + warp) * 32 + lane) * 16) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
    sum += __shfl_xor_sync(kFull, sum, 1);
    sum += __shfl_xor_sync(kFull, sum, 2);
    if (t == 0) {
      s_qs[warp * 8 + g] = kInt8 ? up * kTwo24 : up;
      s_qb[warp * 8 + g] = kInt8 ? -128.f * sum * up : 0.f;
    }
  }
  __syncthreads();
  float qs[NB][2], qb[NB][2];  // of rows 2 t, 2 t + 1
  int lim[NB][2];              // their visible keys
  uint4 qr[NB == 1 ? KS / 2 : 1];
  if constexpr (NB == 1) {
#pragma unroll
    for (int i = 0; i < KS / 2; ++i) qr[i] = lds16(qf + (i * 32 + lane) * 16);
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = nb * 8 + 2 * t + i;
      qs[nb][i] = s_qs[r];
      qb[nb][i] = s_qb[r];
      lim[nb][i] = first_row + r < rows ? start + (first_row + r) / p.G + 1 : 0;
    }
  float* sp = nullptr;         // scores of token g, rows 2 t and on
  if constexpr (MASS) sp = p.ws_s + (item * Lp + g) * p.RS + 2 * t;

  float o[NB][MT][4], ps[NB][4];
  float M[NB][2], l[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int j = 0; j < MT; ++j) o[nb][j][0] = o[nb][j][1] = o[nb][j][2] = o[nb][j][3] = 0.f;
    ps[nb][0] = ps[nb][1] = ps[nb][2] = ps[nb][3] = 0.f;
    M[nb][0] = M[nb][1] = kNone;
    l[nb][0] = l[nb][1] = 0.f;
  }

  for (int j = 0; j < count; j += U) {
    issue(j / U + AHEAD);
    cp_async_wait<AHEAD>();  // this lane's share of pages j .. j + U - 1 has landed
    __syncwarp();
    uint32_t st[U];
    float lv[U], rv[U], s[U][NB][4];
    int key0[U];
    // ---- S^T = K Q^T
#pragma unroll
    for (int u = 0; u < U; ++u) {
      st[u] = ring + ((j + u) % kStages) * PB;
      // past the warp's last page every key is hidden
      key0[u] = j + u < count ? (first + kWarps * (j + u)) * kP8Page : 1 << 30;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        s[u][nb][0] = s[u][nb][1] = s[u][nb][2] = s[u][nb][3] = 0.f;
    }
#pragma unroll
    for (int hh = 0; hh < KH; ++hh) {
      uint4 ka[U], kb[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ka[u] = lds16(st[u] + k_off[hh]);
        kb[u] = lds16(st[u] + k_off[hh] + HALF);
      }
#pragma unroll
      for (int w2 = 0; w2 < 2; ++w2) {
        uint4 qv[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if constexpr (NB == 1)
            qv[nb] = qr[hh * 2 + w2];
          else
            qv[nb] = lds16(qf + (((hh * 2 + w2) * NB + nb) * 32 + lane) * 16);
        }
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int u = 0; u < U; ++u) {
            uint32_t a0, a1, a2, a3;
            operand<FMT>(flip<FMT>(word_of(ka[u], 2 * w2 + w)), a0, a2);
            operand<FMT>(flip<FMT>(word_of(kb[u], 2 * w2 + w)), a1, a3);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              mma_f16(s[u][nb], a0, a1, a2, a3, word_of(qv[nb], 2 * w), word_of(qv[nb], 2 * w + 1));
          }
      }
    }
    // ---- w = s + log2(vs)
    bool edge = false, grow = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = (j + u) & 31;
      const float ks = __shfl_sync(kFull, ks_i, at);
      lv[u] = __shfl_sync(kFull, lv_i, at);
      rv[u] = __shfl_sync(kFull, rv_i, at);
      edge |= key0[u] + kP8Page > min_lim;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float y4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = e & 1;  // row 2 t + i, token g + 8 (e / 2)
          const float y = fmaf(s[u][nb][e], qs[nb][i], qb[nb][i]);
          // one rounding either way, so that the output does not depend on the weights' being kept
          s[u][nb][e] = fmaf(y, ks, lv[u]);
          if constexpr (MASS) y4[e] = y * ks;
        }
        if constexpr (MASS)
          // either row may see no key: the first of them lies before the sequence's first token
          // or the second past the last row
          if (max(lim[nb][0], lim[nb][1]) > 0 && (u == 0 || j + u < count)) {
            float* to = sp + static_cast<int64_t>(key0[u]) * p.RS + nb * 8;
            *reinterpret_cast<float2*>(to) = make_float2(y4[0], y4[1]);
            *reinterpret_cast<float2*>(to + 8 * p.RS) = make_float2(y4[2], y4[3]);
          }
      }
    }
    if (edge) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0[u] + g + 8 * (e >> 1) >= lim[nb][e & 1]) s[u][nb][e] = -INFINITY;
    }
    float mx[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float m = fmaxf(s[0][nb][i], s[0][nb][2 + i]);
        if constexpr (U == 2) m = fmaxf(m, fmaxf(s[U - 1][nb][i], s[U - 1][nb][2 + i]));
        mx[nb][i] = m;
        grow |= m > M[nb][i] + kGrow;
      }
    if (__any_sync(kFull, grow)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float m = mx[nb][i];
          m = fmaxf(m, __shfl_xor_sync(kFull, m, 4));
          m = fmaxf(m, __shfl_xor_sync(kFull, m, 8));
          m = fmaxf(m, __shfl_xor_sync(kFull, m, 16));
          m = fmaxf(m, M[nb][i]);
          const float a = ex2f(M[nb][i] - m);
          M[nb][i] = m;
          l[nb][i] *= a;
          ps[nb][i] *= a;
#pragma unroll
          for (int jj = 0; jj < MT; ++jj) {
            o[nb][jj][i] *= a;
            o[nb][jj][2 + i] *= a;
          }
        }
    }
    uint32_t pb[U][NB][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float rl = fabsf(rv[u]);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float e4[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          e4[i] = ex2f(s[u][nb][i] - M[nb][i]);
          e4[2 + i] = ex2f(s[u][nb][2 + i] - M[nb][i]);
          l[nb][i] = fmaf(e4[i] + e4[2 + i], rl, l[nb][i]);
        }
        pb[u][nb][0] = transpose8x8(half2_of(e4[0], e4[1]));
        pb[u][nb][1] = transpose8x8(half2_of(e4[2], e4[3]));
      }
      if (rv[u] < 0.f) {  // a V block of zeros adds to l alone
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) pb[u][nb][0] = pb[u][nb][1] = 0u;
      }
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t v[4][VW];         // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = st[u] + v_off[i & 1] + (i >> 1) * HALF;
        if constexpr (D == 128) {
          const uint4 x = lds16(a);
#pragma unroll
          for (int w = 0; w < 4; ++w) v[i][w] = flip<FMT>(word_of(x, w));
        } else {
          const uint2 x = lds8(a);
          v[i][0] = flip<FMT>(x.x);
          v[i][1] = flip<FMT>(x.y);
        }
      }
      if constexpr (!kInt8) {  // codes past the last visible key may be NaN
        const int live = n_keys - key0[u];
        if (live < kP8Page) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (2 * t + (i & 1) + 8 * (i >> 1) >= live)
#pragma unroll
              for (int w = 0; w < VW; ++w) v[i][w] = 0u;
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {  // bytes 4 w + 2 hf, + 1 of the piece
          const uint32_t sel = hf == 0 ? 0x5140 : 0x7362;
          uint32_t a0, a1, a2, a3;
          operand<FMT>(__byte_perm(v[0][w], v[1][w], sel), a0, a1);
          operand<FMT>(__byte_perm(v[2][w], v[3][w], sel), a2, a3);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            mma_f16(o[nb][2 * w + hf], a0, a1, a2, a3, pb[u][nb][0], pb[u][nb][1]);
        }
      if constexpr (kInt8) {
        constexpr uint32_t kOnes = 0x3c003c00u;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          mma_f16(ps[nb], kOnes, kOnes, kOnes, kOnes, pb[u][nb][0], pb[u][nb][1]);
      }
    }
    __syncwarp();  // every lane is done with these stages before they are refilled
  }
  cp_async_wait<0>();
  __syncthreads();  // the ring becomes the join's buffer

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
        s_m[warp * R + r] = M[nb][i];
        s_l[warp * R + r] = x;
      }
      const float off = -128.f * ps[nb][i];
      auto val = [&](int j, int z) {
        return kInt8 ? fmaf(o[nb][j][z + i], kTwo24, off) : o[nb][j][z + i];
      };
      // dims g D / 8 + 2 j (+ 1): element j of the lane's piece, two per m-tile
      if (first_row + r < rows) {
#pragma unroll
        for (int j = 0; j < MT; j += 2)
          *reinterpret_cast<float4*>(s_o + (warp * R + r) * D + g * DL + 2 * j) =
              make_float4(val(j, 0), val(j, 2), val(j + 1, 0), val(j + 1, 2));
      }
    }
  __syncthreads();
  const int64_t slot = item * p.splits + split;
  for (int e = threadIdx.x; e < R * (D / 4); e += kWarps * 32) {
    const int r = e / (D / 4), d = (e % (D / 4)) * 4;
    if (first_row + r >= rows) break;
    float m = s_m[r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w * R + r]);
    float den = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float x = ex2f(s_m[w * R + r] - m);
      const float4 y = *reinterpret_cast<const float4*>(s_o + (w * R + r) * D + d);
      den = fmaf(s_l[w * R + r], x, den);
      acc.x = fmaf(y.x, x, acc.x);
      acc.y = fmaf(y.y, x, acc.y);
      acc.z = fmaf(y.z, x, acc.z);
      acc.w = fmaf(y.w, x, acc.w);
    }
    const float inv = den == 0.f ? 0.f : __fdiv_rn(1.f, den);  // no visible key: 0
    acc.x *= inv;
    acc.y *= inv;
    acc.z *= inv;
    acc.w *= inv;
    if (uncut) {
      const int64_t orow = static_cast<int64_t>(si.row0 + (first_row + r) / p.G) * p.Hq +
                           h * p.G + (first_row + r) % p.G;
      uint2 u;
      u.x = P8Io<T>::pack(acc.x, acc.y);
      u.y = P8Io<T>::pack(acc.z, acc.w);
      *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + orow * D + d) = u;
    } else {
      *reinterpret_cast<float4*>(p.ws_o + (slot * R + r) * D + d) = acc;
    }
    if (d == 0 && (MASS || !uncut)) {
      const float lse = den == 0.f ? -INFINITY : m + log2f(den);
      if (MASS && p.splits == 1 && p.row_tiles == 1)
        s_qs[r] = lse;
      else
        p.ws_lse[slot * R + r] = lse;
    }
  }
  if constexpr (MASS) {
    if (p.splits == 1 && p.row_tiles == 1) {  // this CTA has every row and key of the head
      __syncthreads();
      for (int j = threadIdx.x; j < si.kv; j += kWarps * 32) {
        const int64_t at = mass_at(p, table, h, j);
        p.mass_out[at] = p.mass_in[at] + weight_of<R>(p.ws_s + (item * Lp + j) * p.RS, 0,
                                                      max(0, j - start) * p.G, rows, s_qs);
      }
    }
  }
}

// Joins the chunks of an item: out = sum 2^(lse_c - L) o_c with L = log2 sum 2^lse_c, in the
// order of its pages.  `wpr` warps share a row (eight where there are many chunks).  With
// mass, further CTAs of kTokens tokens of a (sequence, KV head) add the weights.  Launched so
// that its start overlaps the end of p8_attn_kernel, which it waits for.
constexpr int kTokens = 1024;
template <typename T, int D, int NB, bool MASS>
__global__ void __launch_bounds__(256)
    p8_finish_kernel(const AttnParams p, int join_ctas, int wpr) {
  constexpr int R = 8 * NB;
  constexpr int VL = D / 32;  // dims of a lane
  __shared__ float s_lse[kP8ShortRows];
  __shared__ float s_acc[8][D];
  const int seq = blockIdx.y / p.c.Hkv, h = blockIdx.y % p.c.Hkv;
  const SeqInfo si = seq_info(p, seq);  // inputs, complete before p8_attn_kernel began
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int start = si.kv - si.q_len;
  const int64_t item0 = static_cast<int64_t>(blockIdx.y) * p.row_tiles;
  auto chunks_of = [&](int rt) {
    const int last_tok = (min(si.rows, (rt + 1) * R) - 1) / p.G;
    const int n_pages = (max(0, start + last_tok + 1) + kP8Page - 1) / kP8Page;
    return max(1, (n_pages + p.chunk - 1) / p.chunk);
  };
  // a row's L, by one warp
  auto total_lse = [&](const float* lse, int n) {
    float m = -INFINITY;
    for (int c = lane; c < n; c += 32) m = fmaxf(m, lse[c * R]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
    const float base = m == -INFINITY ? 0.f : m;
    float den = 0.f;
    for (int c = lane; c < n; c += 32) den += ex2f(lse[c * R] - base);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(kFull, den, o);
    return den == 0.f ? -INFINITY : base + log2f(den);
  };
  const int j0 = (static_cast<int>(blockIdx.x) - join_ctas) * kTokens;
  int64_t at[kTokens / 256];
  float before[kTokens / 256];
  if constexpr (MASS) {  // the masses so far are inputs as well
#pragma unroll
    for (int i = 0; i < kTokens / 256; ++i) {
      const int j = j0 + i * 256 + threadIdx.x;
      if (j0 >= 0 && j < si.kv) {
        at[i] = mass_at(p, p.s.table + static_cast<int64_t>(seq) * p.s.max_pages, h, j);
        before[i] = p.mass_in[at[i]];
      }
    }
  }
  p8_grid_wait();
  if (static_cast<int>(blockIdx.x) < join_ctas) {
    const int rr = (blockIdx.x * 8 + warp) / wpr, part = warp % wpr;
    const int rt = rr / R, r = rr % R;
    const int n = rr < si.rows ? chunks_of(rt) : 0;
    float acc[VL] = {};
    if (n > 1) {
      const int64_t slot = (item0 + rt) * p.splits;
      const float* lse = p.ws_lse + slot * R + r;
      const float* src = p.ws_o + (slot * R + r) * D + lane * VL;
      // four chunks at a time, the first four before L is known
      float x[4][VL], ls[4];
      auto fetch = [&](int c0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = c0 + k * wpr;
          if (c >= n) break;
          ls[k] = lse[c * R];
          if constexpr (VL == 4)
            *reinterpret_cast<float4*>(x[k]) =
                *reinterpret_cast<const float4*>(src + static_cast<int64_t>(c) * R * D);
          else
            *reinterpret_cast<float2*>(x[k]) =
                *reinterpret_cast<const float2*>(src + static_cast<int64_t>(c) * R * D);
        }
      };
      fetch(part);
      float L = total_lse(lse, n);
      if (L == -INFINITY) L = 0.f;
      for (int c0 = part; c0 < n; c0 += 4 * wpr) {
        if (c0 != part) fetch(c0);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (c0 + k * wpr >= n) break;
          const float w = ex2f(ls[k] - L);
#pragma unroll
          for (int i = 0; i < VL; ++i) acc[i] = fmaf(w, x[k][i], acc[i]);
        }
      }
    }
    if (wpr > 1) {  // all eight warps have one row
#pragma unroll
      for (int i = 0; i < VL; ++i) s_acc[warp][lane * VL + i] = acc[i];
      __syncthreads();
      if (warp > 0) return;
#pragma unroll
      for (int i = 0; i < VL; ++i)
        for (int w = 1; w < 8; ++w) acc[i] += s_acc[w][lane * VL + i];
    }
    if (n > 1) {
      const int64_t orow = static_cast<int64_t>(si.row0 + rr / p.G) * p.Hq + h * p.G + rr % p.G;
      uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + orow * D + lane * VL);
#pragma unroll
      for (int i = 0; i < VL; i += 2) dst[i / 2] = P8Io<T>::pack(acc[i], acc[i + 1]);
    }
    return;
  }
  if constexpr (MASS) {
    if (j0 >= si.kv) return;
    for (int r = warp; r < si.rows; r += 8) {
      const float L = total_lse(p.ws_lse + (item0 + r / R) * p.splits * R + r % R, chunks_of(r / R));
      if (lane == 0) s_lse[r] = L;
    }
    __syncthreads();
    const int64_t Lp = static_cast<int64_t>(p.s.max_pages) * kP8Page;
#pragma unroll
    for (int i = 0; i < kTokens / 256; ++i) {
      const int j = j0 + i * 256 + threadIdx.x;
      if (j < si.kv)
        p.mass_out[at[i]] = before[i] + weight_of<R>(p.ws_s + (item0 * Lp + j) * p.RS,
                                                     Lp * p.RS, max(0, j - start) * p.G, si.rows,
                                                     s_lse);
    }
  }
}

// Joins the splits of a long chunk's rows: out = sum 2^(lse_s - L) o_s with
// L = log2 sum 2^lse_s, which goes to `total` where the weights need it.  A thread has four
// dims of a row; all it reads is on its way before it is looked at.  Rows outside
// [cu_q[0], cu_q[S]) are other calls': their part of the workspace was never written, and
// their outputs stay.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    p8_combine_kernel(const float* __restrict__ ws_o, const float* __restrict__ ws_lse,
                      float* __restrict__ total, T* __restrict__ out, P8Seqs seqs, int Hq,
                      int64_t rows, int splits) {
  constexpr int kMost = 4;  // splits read ahead
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = at / (D / 4);
  const int d = static_cast<int>(at % (D / 4)) * 4;
  // inputs, complete before the chunk kernel began
  const int64_t begin = static_cast<int64_t>(__ldg(seqs.cu_q)) * Hq;
  const int64_t end = static_cast<int64_t>(__ldg(seqs.cu_q + seqs.num_seqs)) * Hq;
  p8_grid_wait();
  if (row >= rows || row < begin || row >= end) return;
  const float* lse = ws_lse + row * splits;
  const float* o = ws_o + row * splits * D + d;
  float ls[kMost];
  float4 x[kMost];
#pragma unroll
  for (int s = 0; s < kMost; ++s)
    if (s < splits) {
      ls[s] = lse[s];
      x[s] = *reinterpret_cast<const float4*>(o + s * D);
    }
  float m = -INFINITY;
#pragma unroll
  for (int s = 0; s < kMost; ++s)
    if (s < splits) m = fmaxf(m, ls[s]);
  for (int s = kMost; s < splits; ++s) m = fmaxf(m, lse[s]);
  const float base = m == -INFINITY ? 0.f : m;
  float den = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float l, const float4& y) {
    const float w = ex2f(l - base);
    if (w == 0.f) return;  // a split without keys of this row left nothing to read
    den += w;
    acc.x = fmaf(w, y.x, acc.x);
    acc.y = fmaf(w, y.y, acc.y);
    acc.z = fmaf(w, y.z, acc.z);
    acc.w = fmaf(w, y.w, acc.w);
  };
#pragma unroll
  for (int s = 0; s < kMost; ++s)
    if (s < splits) add(ls[s], x[s]);
  for (int s = kMost; s < splits; ++s) add(lse[s], *reinterpret_cast<const float4*>(o + s * D));
  const float inv = den == 0.f ? 0.f : __fdiv_rn(1.f, den);
  uint2 u;
  u.x = P8Io<T>::pack(acc.x * inv, acc.y * inv);
  u.y = P8Io<T>::pack(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(out + row * D + d) = u;
  if (total != nullptr && d == 0) total[row] = den == 0.f ? -INFINITY : base + log2f(den);
}

template <typename T, int FMT, int D, int NB, bool MASS>
int launch_nb(const AttnParams& p, cudaStream_t st) {
  using Cfg = AttnCfg<D, NB>;
  constexpr auto kern = p8_attn_kernel<T, FMT, D, NB, MASS>;
  int rc = p8_opt_in<kern>(Cfg::SMEM);
  if (rc) return rc;
  rc = p8_launch(kern, dim3(p.splits * p.row_tiles, p.c.Hkv, p.s.num_seqs), kWarps * 32, Cfg::SMEM,
                 st, p);
  if (rc || (p.splits == 1 && !(MASS && p.row_tiles > 1))) return rc;
  const int wpr = p.splits > 16 ? 8 : 1;
  const int join = p.splits > 1 ? p.row_tiles * NB * wpr : 0;
  const int tokens = MASS ? (p.s.max_pages * kP8Page + kTokens - 1) / kTokens : 0;
  return p8_launch(p8_finish_kernel<T, D, NB, MASS>, dim3(join + tokens, p.c.Hkv * p.s.num_seqs),
                   256, 0, st, p, join, wpr);
}

template <typename T, int FMT, int D>
int launch_attn(const AttnParams& p, int nb, cudaStream_t st) {
  const bool mass = p.mass_out != nullptr;
#define CFB_NB(NBV)                                                       \
  case NBV:                                                               \
    return mass ? launch_nb<T, FMT, D, NBV, true>(p, st)            \
                : launch_nb<T, FMT, D, NBV, false>(p, st);
  switch (nb) {
    CFB_NB(1)
    CFB_NB(2)
    CFB_NB(3)
    CFB_NB(4)
    default: return -2;
  }
#undef CFB_NB
}

}  // namespace

int p8_combine(const P8Seqs& s, const P8Attn& a, int D, cudaStream_t st) {
  const int64_t n = a.N * a.Hq;
  const int64_t grid = (n * (D / 4) + 255) / 256;
  if (grid > 0x7fffffff) return -3;
  const dim3 g(static_cast<unsigned>(grid));
#define CFB_COMBINE(T, DD)                                                                  \
  return p8_launch(p8_combine_kernel<T, DD>, g, 256, 0, st, a.ws_o, a.ws_lse, a.ws_total,   \
                   static_cast<T*>(a.out), s, a.Hq, n, a.splits)
  if (a.type == kP8Bf16) {
    if (D == 128) CFB_COMBINE(__nv_bfloat16, 128);
    CFB_COMBINE(__nv_bfloat16, 64);
  }
  if (D == 128) CFB_COMBINE(__half, 128);
  CFB_COMBINE(__half, 64);
#undef CFB_COMBINE
}

P8AttnPlan p8_attn_plan(const P8Cache& c, const P8Seqs& s, int group, int max_q_len, bool mass,
                        int num_sms) {
  P8AttnPlan pl;
  const int rows = max_q_len * group;
  // as few row tiles as 32 rows of a CTA allow: a tile reads and converts all its pages
  pl.row_tiles = (rows + 31) / 32;
  pl.nb = ((rows + pl.row_tiles - 1) / pl.row_tiles + 7) / 8;
  const int64_t items = static_cast<int64_t>(s.num_seqs) * c.Hkv * pl.row_tiles;
  const int R = 8 * pl.nb;
  if (s.max_pages <= kWholePages) {
    pl.chunk = kWholePages;
  } else {  // about three waves of CTAs, were all sequences as long as the table is wide;
    // 64 ragged requests: 38 us so, 44 with 16 to 32 pages and eight waves, 45 with 64 to 128 and
    // one (one request of 131072 tokens, 8/1 heads: 18.7, 27.1 and 17.0)
    const int64_t ctas = 3 * static_cast<int64_t>(num_sms) * (pl.nb <= 2 ? 3 : 2);
    const int64_t chunk = (items * s.max_pages + ctas - 1) / ctas;
    pl.chunk = static_cast<int>(std::min<int64_t>(std::max<int64_t>(chunk, kMinPages), kMaxPages));
  }
  pl.splits = (s.max_pages + pl.chunk - 1) / pl.chunk;
  if (pl.splits > 1) pl.n_o = items * pl.splits * R * c.D;
  if (pl.splits > 1 || mass) pl.n_lse = items * pl.splits * R;
  pl.score_rows = rows <= 4 ? 4 : R;
  if (mass) pl.n_s = items * pl.score_rows * s.max_pages * kP8Page;
  return pl;
}

int p8_attention(const P8Cache& c, const P8Seqs& s, const P8Attn& a, const P8AttnPlan& plan,
                 float* ws, int* err, cudaStream_t stream) {
  if (s.num_seqs <= 0) return 0;
  const int64_t heads = static_cast<int64_t>(s.num_seqs) * c.Hkv;
  if (heads > 65535 || c.num_pages * c.Hkv > 0x7fffffff ||
      static_cast<int64_t>(plan.splits) * plan.row_tiles > 0x7fffffff ||
      plan.chunk > 32 * kWarps || static_cast<int64_t>(a.max_q_len) * (a.Hq / c.Hkv) > kP8ShortRows)
    return -3;
  AttnParams p;
  p.c = c;
  p.s = s;
  p.q = a.q;
  p.q_stride = a.q_stride;
  p.out = a.out;
  p.N = a.N;
  p.Hq = a.Hq;
  p.G = a.Hq / c.Hkv;
  p.row_tiles = plan.row_tiles;
  p.max_rows = a.max_q_len * p.G;
  p.chunk = plan.chunk;
  p.splits = plan.splits;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.ws_o = ws;
  p.ws_lse = p.ws_o + plan.n_o;
  p.ws_s = p.ws_lse + plan.n_lse;
  p.RS = plan.score_rows;
  p.mass_in = a.mass_in;
  p.mass_out = a.mass_out;
  p.err = err;
  int rc = 0;
  switch (a.type * 4 + c.fmt * 2 + (c.D == 128)) {
    case 0: rc = launch_attn<__nv_bfloat16, kP8Int8, 64>(p, plan.nb, stream); break;
    case 1: rc = launch_attn<__nv_bfloat16, kP8Int8, 128>(p, plan.nb, stream); break;
    case 2: rc = launch_attn<__nv_bfloat16, kP8E4m3, 64>(p, plan.nb, stream); break;
    case 3: rc = launch_attn<__nv_bfloat16, kP8E4m3, 128>(p, plan.nb, stream); break;
    case 4: rc = launch_attn<__half, kP8Int8, 64>(p, plan.nb, stream); break;
    case 5: rc = launch_attn<__half, kP8Int8, 128>(p, plan.nb, stream); break;
    case 6: rc = launch_attn<__half, kP8E4m3, 64>(p, plan.nb, stream); break;
    case 7: rc = launch_attn<__half, kP8E4m3, 128>(p, plan.nb, stream); break;
    default: return -2;
  }
  return rc ? rc : static_cast<int>(cudaGetLastError());
}

}  // namespace cfb
