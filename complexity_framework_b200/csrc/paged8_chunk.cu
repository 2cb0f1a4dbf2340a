// Attention over the 8-bit paged KV cache (sm_100a): long chunks of new tokens.
//
// With hundreds of rows (new tokens x grouped heads) for each KV head the work is bound by
// the tensor cores and by exponentials, not by the cache's bytes, so it goes to tcgen05.
// Every CTA of a KV head needs the same keys and values as 16-bit operands.  Converting
// them in each CTA costs about as many instruction slots as its softmax; they are expanded
// once instead, into a workspace that TMA reads back from L2:
//   K as its codes in q's type, V as its codes in f16: both exact.  The block scales stay
//   in fp32 and cost nothing: K's multiplies the softmax scale, log2 of V's is added in the
//   exponent, so that P carries it (w = s + log2 vs, P = 2^(w - M), l = sum P / vs; see
//   paged8_attn.cu), and P is rounded to f16.
//
// p8_chunk_kernel: one CTA per (NQ x 128 rows, KV head, sequence, KV split).  A row tile
// packs floor(128 / G) tokens x G heads, so all the heads of a group share each K/V tile.
//   warps 0 .. 4 NQ - 1  softmax, one row per thread: S from TMEM, P against a bound that
//                        moves only when f16 would overflow, P back to TMEM
//   next warp            TMA producer: Q once, then K and V tiles through rings of their own
//   last warp            MMA issuer: S_x = Q_x K^T of the next tile, then O_x += P_x V
// Key tiles are 64 wide so that TMEM (512 columns) holds two S of each row tile beside O:
// the next S is there when a softmax warp ends a tile.  With 128-wide tiles and one S the
// chain S -> P -> O -> S left the softmax warps idle for 40% of a tile (4100 cycles for 128
// keys of two row tiles, of which their exponentials need 2100).  A cubic on the FMA pipe for
// a share of the exponentials was not worth its code (140.9 us with a quarter of them, 142.8
// without, before later changes).
// Measured: 2 x 1024 tokens over 3077 and 5120, GQA 32/8, D 128: 146 us with the expansion (12),
// 825 TFLOP/s, tensor pipe 45% and exponential unit 46% busy; neither is the limit, likely the
// softmax warps' waits.  Half a row a thread (twice the warps) was slower: 159 us against 144.
// p8_chunk_mass_kernel: weights summed over the rows need each row's final log-sum-exp, so
// they are recomputed: one CTA per (128 keys, KV head, sequence) walks the row tiles with
// S^T = K Q^T (a thread owns a key), adding 2^(s - lse) in a fixed order: no atomics, the same
// bits every time.  Where that leaves SMs idle a cluster shares the row tiles of a key tile
// and its first CTA adds the others' sums up over distributed shared memory.
#include <type_traits>

#include "paged8.cuh"

#include "flash.h"

namespace cfb {
namespace {

constexpr int kT = 128;               // rows of a tile
constexpr int kKeys = 64;             // keys of a tile of the forward kernel
constexpr float kMostSum = 8192.f;    // of a row's P in a key tile: no P overflows f16
constexpr float kTinyScale = 7.888609e-31f;  // 2^-100: blocks below it count as zeros

__device__ __forceinline__ float ex2c(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// kind::f16 instruction descriptor, fp32 accumulators: A and B both bf16 or both f16.
template <typename T>
__host__ __device__ constexpr uint32_t idesc16(int M, int N, bool b_mn) {
  return (1u << 4) | (sizeof(T) == 2 && P8Io<T>::kBf16 ? (1u << 7) | (1u << 10) : 0u) |
         ((b_mn ? 1u : 0u) << 16) | ((static_cast<uint32_t>(N) >> 3) << 17) |
         ((static_cast<uint32_t>(M) >> 4) << 24);
}

__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > kWaitBoundNs) return;
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                          int* err, int code, int site) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, code, site));
}

// 16 columns of TMEM into registers, and the wait that makes them readable: the registers
// pass through the wait, so no use of them can move before it.
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// After a wait: no use of these registers can move before this point.
__device__ __forceinline__ void tmem_ready32(uint32_t (&r)[32]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}

// ---------------------------------------------------------------------------- expand
// One warp per (sequence, block, head, K or V) of the workspace
//   k_ws, v_ws [S, Hkv, Lw, D],  par [S, Hkv, Lw / 16],  Lw a multiple of 128,
// where par holds (ks * scale * log2 e, log2 vs, 1 / vs) of a block.  Tokens past the
// sequence, up to the end of its last 128-key tile, become zeros.  A block whose V scale is
// not finite gets V = 0 and a NaN K scale: the rows that see the block read NaN, and the rows
// that do not are not reached by 0 * NaN.  A scale of (nearly) zero becomes zero codes with a
// harmless scale: 1 for K, so that no masked score meets -inf * 0, and 2^-24 for V, so that
// the block does not raise the bound of w.
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(256)
    p8_expand_kernel(P8Cache c, P8Seqs s, int blocks, unsigned units, float scale_log2,
                     T* __restrict__ k_ws, __half* __restrict__ v_ws, float4* __restrict__ par,
                     int* err) {
  constexpr int NC = kP8Page * D / 8 / 32;
  const unsigned unit = blockIdx.x * 8 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int x = unit & 1, h = (unit >> 1) % c.Hkv, blk = (unit >> 1) / c.Hkv;
  const int seq = blockIdx.y;
  p8_grid_wait();
  if (unit >= units) return;
  const int entry = __ldg(s.table + static_cast<int64_t>(seq) * s.max_pages +
                          min(blk, s.max_pages - 1));
  const int kv = p8_len(s.kv_lens, seq, s.max_pages, err, 80);
  if (blk * kP8Page >= (kv + kT - 1) / kT * kT) return;
  const int64_t sh = static_cast<int64_t>(seq) * c.Hkv + h;
  int live = min(kv - blk * kP8Page, kP8Page);
  uint4* dst = reinterpret_cast<uint4*>(
      (x ? reinterpret_cast<uint16_t*>(v_ws) : reinterpret_cast<uint16_t*>(k_ws)) +
      (sh * blocks + blk) * (kP8Page * D));
  const uint8_t* src = nullptr;
  float4 f = make_float4(scale_log2, -24.f, 16777216.f, 0.f);
  if (live > 0) {
    const int64_t page = p8_checked(entry, c.num_pages, err, 81);
    const int64_t ph = page * c.Hkv + h;
    const float2 sc = __ldg(reinterpret_cast<const float2*>(c.scales) + ph);
    const bool fine = fabsf(sc.y) <= 3.402823466e38f;
    if (!(sc.x < kTinyScale)) f.x = sc.x * scale_log2;
    if (!fine) f.x = __uint_as_float(0x7fc00000u);
    if (fine && sc.y >= kTinyScale) {
      f.y = log2f(sc.y);
      f.z = __fdiv_rn(1.f, sc.y);
    }
    if (x == 0 ? sc.x < kTinyScale : !fine || sc.y < kTinyScale) live = 0;
    src = c.codes + (ph * 2 + x) * (kP8Page * D);
  }
  if (x == 0 && lane == 0) par[sh * blocks + blk] = f;
  uint2 w[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int e = (i * 32 + lane) * 8;
    w[i] = e / D < live ? __ldg(reinterpret_cast<const uint2*>(src + e)) : make_uint2(0, 0);
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    uint32_t o[4] = {};
    if ((i * 32 + lane) * 8 / D < live) {
      p8_to_half<FMT>(w[i].x, o[0], o[1]);
      p8_to_half<FMT>(w[i].y, o[2], o[3]);
      if (P8Io<T>::kBf16 && x == 0) {
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const float2 v = __half22float2(*reinterpret_cast<__half2*>(&o[z]));
          o[z] = pack_bf16x2(v.x, v.y);
        }
      }
    }
    dst[i * 32 + lane] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// --------------------------------------------------------------------------- forward
struct ChunkParams {
  const int32_t* cu_q;
  const int32_t* kv_lens;
  int max_pages, blocks;       // page-table width; workspace blocks of a sequence
  const float4* par;           // block scales of the workspace
  void* out;
  float* lse;                  // [N * Hq, splits], log2 units (splits > 1, or for the weights)
  float* ws_o;                 // [N * Hq, splits, D] (splits > 1)
  int64_t N;
  int Hq, Hkv, G, splits, row_ctas, num_seqs, max_q_len;
  int* err;
};

template <int D, int NQ>
struct ChunkCfg {
  static constexpr int STAGES = NQ == 1 && D == 128 ? 2 : 4;  // of K, and of V
  static constexpr int CTAS = NQ == 1 ? 2 : 1;        // on an SM
  static constexpr int CHUNKS = D / 64;
  static constexpr int Q_BYTES = kT * D * 2;
  static constexpr int K_BYTES = kKeys * D * 2;
  static constexpr int BLOCKS = kKeys / kP8Page;      // scale blocks of a key tile
  static constexpr int SOFT = 4 * NQ;                 // softmax warps
  static constexpr int SMEM =
      NQ * Q_BYTES + STAGES * 2 * K_BYTES + 1024 + 512 + SOFT * 2 * BLOCKS * 16;
  static constexpr uint32_t T_O = NQ * 2 * kKeys;     // two S of each row tile, then O
  static constexpr uint32_t TMEM = T_O + NQ * D <= 256 ? 256 : 512;
  static constexpr int PRODUCER = SOFT, MMA = SOFT + 1;
  static constexpr int THREADS = (SOFT + 2) * 32;
  static_assert(T_O + NQ * D <= TMEM, "TMEM budget");
  static_assert(CTAS * (SMEM + 1024) <= 233472, "shared memory");
};

struct alignas(16) ChunkBars {
  uint64_t q_full;
  uint64_t k_full[4], k_empty[4];
  uint64_t v_full[4], v_empty[4];
  uint64_t s_full[2][2];   // [row tile][S buffer]
  uint64_t p_full[2][2];
  uint64_t o_full[2][2];   // O += P V; two, as the next may be done before this one is awaited
  uint64_t mma_done;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(ChunkBars) % 16 == 0 && sizeof(ChunkBars) <= 512, "block scales follow");

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(ChunkCfg<D, NQ>::THREADS, (ChunkCfg<D, NQ>::CTAS))
    p8_chunk_kernel(const __grid_constant__ CUtensorMap tmQ,
                    const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const ChunkParams p) {
  using Cfg = ChunkCfg<D, NQ>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + NQ * Cfg::Q_BYTES;
  uint8_t* sV = sK + STAGES * Cfg::K_BYTES;
  ChunkBars* bars = reinterpret_cast<ChunkBars*>(sV + STAGES * Cfg::K_BYTES);
  volatile int* abort_flag = &bars->abort;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  // The most work first, so that no long CTA starts late: the longest sequence (of the first
  // 32; more of them even out by themselves), and in it the last row tiles, which see the
  // most keys.
  const unsigned each = p.splits * p.Hkv * p.row_ctas;
  int seq = static_cast<int>(blockIdx.x / each);
  const int rest = static_cast<int>(blockIdx.x % each);
  const int rc = p.row_ctas - 1 - rest / (p.splits * p.Hkv);
  const int split = rest % p.splits, h = rest / p.splits % p.Hkv;
  if (p.num_seqs <= 32) {
    const int len = lane < p.num_seqs ? __ldg(p.kv_lens + lane) : -1;
    int rank = 0;
    for (int i = 0; i < p.num_seqs; ++i) {
      const int other = __shfl_sync(0xffffffffu, len, i);
      rank += other > len || (other == len && i < lane);
    }
    seq = __ffs(__ballot_sync(0xffffffffu, lane < p.num_seqs && rank == seq)) - 1;
  }
  const int row0 = __ldg(p.cu_q + seq), q_len = __ldg(p.cu_q + seq + 1) - row0;
  if (row0 < 0 || q_len < 0 || static_cast<int64_t>(row0) + q_len > p.N) {
    if (threadIdx.x == 0) report_error(p.err, kErrBounds, 82);
    p8_grid_wait();  // no CTA ends before the kernels it follows
    return;
  }
  const int kv = p8_len(p.kv_lens, seq, p.max_pages, p.err, 83);
  const int TT = kT / p.G;                 // tokens of a row tile
  const int tok0 = rc * NQ * TT;
  if (q_len > p.max_q_len && threadIdx.x == 0) report_error(p.err, kErrBounds, 84);
  if (tok0 >= q_len) {
    p8_grid_wait();
    return;
  }
  const int start = kv - q_len;
  // key tiles of row tile x, and this split's share of them
  auto tiles_of = [&](int x) {
    const int t0 = tok0 + x * TT;
    if (t0 >= q_len) return 0;
    const int last = min(q_len, t0 + TT) - 1;
    return (max(0, start + last + 1) + kKeys - 1) / kKeys;
  };
  int tiles = 0;
#pragma unroll
  for (int x = 0; x < NQ; ++x) tiles = max(tiles, tiles_of(x));
  const int per = (tiles + p.splits - 1) / p.splits;
  const int j0 = split * per;
  auto nkv_of = [&](int x) { return max(0, min(tiles_of(x), j0 + per) - j0); };
  int nkv = 0;
#pragma unroll
  for (int x = 0; x < NQ; ++x) nkv = max(nkv, nkv_of(x));
  const int64_t sh = static_cast<int64_t>(seq) * p.Hkv + h;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], 1);
    }
    for (int x = 0; x < NQ; ++x) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bars->s_full[x][b], 1);
        mbar_init(&bars->p_full[x][b], 4);
        mbar_init(&bars->o_full[x][b], 1);
      }
    }
    mbar_init(&bars->mma_done, 1);
    bars->abort = 0;
    fence_barrier_init();
  }
  {  // rows of a tile past its TT * G are no token's: zeros
    const int used = TT * p.G;
    const int rows = kT - used;
    for (int i = threadIdx.x; i < NQ * Cfg::CHUNKS * rows * 8; i += blockDim.x) {
      const int t = i / (rows * 8), r = i % (rows * 8);
      *reinterpret_cast<uint4*>(sQ + t * (kT * 128) + used * 128 + r * 16) =
          make_uint4(0, 0, 0, 0);
    }
    if (rows > 0) fence_proxy_async_shared();
  }
  if (warp == Cfg::MMA) tmem_alloc(&bars->tmem, Cfg::TMEM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  p8_grid_wait();  // the setup above overlaps the expansion's end

  if (warp == Cfg::PRODUCER) {
    if (nkv > 0 && elect_one()) {
      int live = 0;
#pragma unroll
      for (int x = 0; x < NQ; ++x) live += nkv_of(x) > 0;
      mbar_arrive_expect_tx(&bars->q_full, live * Cfg::CHUNKS * TT * p.G * 128);
#pragma unroll
      for (int x = 0; x < NQ; ++x)
        if (nkv_of(x) > 0)
#pragma unroll
          for (int c = 0; c < Cfg::CHUNKS; ++c)
            tma_load_4d(sQ + x * Cfg::Q_BYTES + c * kT * 128, &tmQ, &bars->q_full, c * 64, 0, h,
                        row0 + tok0 + x * TT);
      // K runs one tile ahead: a K stage is free once the tile's scores are computed
      int issued_k = 0, issued_v = 0;
      auto load = [&](int j, const CUtensorMap* map, uint8_t* tiles, uint64_t* full,
                      uint64_t* empty, int& issued) -> bool {
        if (j >= nkv) return true;
        const int st = j % STAGES;
        if (!mbar_wait(&empty[st], ((j / STAGES) & 1) ^ 1, abort_flag, p.err, kErrTimeoutEmpty, 85))
          return false;
        mbar_arrive_expect_tx(&full[st], Cfg::K_BYTES);
#pragma unroll
        for (int c = 0; c < Cfg::CHUNKS; ++c)
          tma_load_4d(tiles + st * Cfg::K_BYTES + c * kKeys * 128, map, &full[st], c * 64,
                      (j0 + j) * kKeys, h, seq);
        ++issued;
        return true;
      };
      bool ok = load(0, &tmK, sK, bars->k_full, bars->k_empty, issued_k);
      for (int j = 0; j < nkv && ok; ++j)
        ok = load(j + 1, &tmK, sK, bars->k_full, bars->k_empty, issued_k) &&
             load(j, &tmV, sV, bars->v_full, bars->v_empty, issued_v);
      drain(&bars->q_full, 0);
      for (int j = issued_k - STAGES < 0 ? 0 : issued_k - STAGES; j < issued_k; ++j)
        drain(&bars->k_full[j % STAGES], (j / STAGES) & 1);
      for (int j = issued_v - STAGES < 0 ? 0 : issued_v - STAGES; j < issued_v; ++j)
        drain(&bars->v_full[j % STAGES], (j / STAGES) & 1);
    }
  } else if (warp == Cfg::MMA) {
    if (nkv > 0 && elect_one()) {
      constexpr uint32_t IDESC_S = idesc16<T>(kT, kKeys, false);
      constexpr uint32_t IDESC_PV = idesc16<__half>(kT, D, true);
      int nkv_x[NQ];
#pragma unroll
      for (int x = 0; x < NQ; ++x) nkv_x[x] = nkv_of(x);
      // S_x(j) = Q_x K_j^T into buffer j & 1: its P_x(j - 2) was consumed by an MMA issued before
      auto issue_s = [&](int j) -> bool {
        if (j >= nkv) return true;
        const int st = j % STAGES;
        if (!mbar_wait(&bars->k_full[st], (j / STAGES) & 1, abort_flag, p.err, kErrTimeoutFull, 88))
          return false;
        tc_fence_after();
        const uint32_t k_base = smem_u32(sK + st * Cfg::K_BYTES);
#pragma unroll
        for (int x = 0; x < NQ; ++x) {
          if (j >= nkv_x[x]) continue;
          const uint32_t q_base = smem_u32(sQ + x * Cfg::Q_BYTES);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_bf16(tmem + (2 * x + (j & 1)) * kKeys,
                      sw128_desc(q_base + (kk >> 2) * (kT * 128) + (kk & 3) * 32, 16, 1024),
                      sw128_desc(k_base + (kk >> 2) * (kKeys * 128) + (kk & 3) * 32, 16, 1024),
                      IDESC_S, kk != 0 ? 1u : 0u);
          umma_commit(&bars->s_full[x][j & 1]);
        }
        umma_commit(&bars->k_empty[st]);
        return true;
      };
      bool ok = mbar_wait(&bars->q_full, 0, abort_flag, p.err, kErrTimeoutFull, 86);
      if (ok) {
        tc_fence_after();
        ok = issue_s(0);
      }
      for (int j = 0; j < nkv && ok; ++j) {
        const int st = j % STAGES;
        ok = issue_s(j + 1) && mbar_wait(&bars->v_full[st], (j / STAGES) & 1, abort_flag, p.err,
                                         kErrTimeoutFull, 79);
        if (!ok) break;
        const uint32_t v_base = smem_u32(sV + st * Cfg::K_BYTES);
#pragma unroll
        for (int x = 0; x < NQ; ++x) {
          if (j >= nkv_x[x]) continue;
          if (!mbar_wait(&bars->p_full[x][j & 1], (j >> 1) & 1, abort_flag, p.err, kErrTimeoutFull,
                         87)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            umma_bf16_ts(tmem + Cfg::T_O + x * D, tmem + (2 * x + (j & 1)) * kKeys + kk * 8,
                         sw128_desc(v_base + kk * 2048, kKeys * 128, 1024), IDESC_PV,
                         (j > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&bars->o_full[x][j & 1]);
        }
        if (ok) umma_commit(&bars->v_empty[st]);
      }
      umma_commit(&bars->mma_done);
      drain(&bars->mma_done, 0);
    }
  } else {
    const int x = warp >> 2, wq = warp & 3;
    const int r = wq * 32 + lane;
    const int tok = tok0 + x * TT + r / p.G;
    const bool mine = r < TT * p.G && tok < q_len;
    const int lim = mine ? start + tok + 1 : 0;   // keys this row sees
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t t_o = tmem + Cfg::T_O + x * D + lane_off;
    const int n = nkv_of(x);
    constexpr int BL = Cfg::BLOCKS;
    const float4* par = p.par + sh * p.blocks + j0 * BL;
    // the tiles' block scales, through this warp's own corner of shared memory: an
    // asynchronous copy one tile ahead, for which no register waits
    float4* s_par2 = reinterpret_cast<float4*>(bars + 1) + warp * (2 * BL);
    auto fetch_par = [&](int j) {
      if (j < n && lane < BL)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(
                         smem_u32(s_par2 + (j & 1) * BL + lane)),
                     "l"(par + j * BL + lane)
                     : "memory");
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // rows that are no token's never see a key and never ask for a rescale
    float m_used = mine ? -INFINITY : 0.f, l = 0.f;
    bool ok = true;
    fetch_par(0);
    for (int j = 0; j < n && ok; ++j) {
      if (!wait_warp(&bars->s_full[x][j & 1], (j >> 1) & 1, abort_flag, p.err, kErrTimeoutTmem,
                     89)) {
        ok = false;
        break;
      }
      tc_fence_after();
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
      const float4* s_par = s_par2 + (j & 1) * BL;
      fetch_par(j + 1);
      const uint32_t t_s = tmem + (2 * x + (j & 1)) * kKeys + lane_off;
      const int kmax = lim - (j0 + j) * kKeys;  // keys of the tile that this row sees
      const bool edge = __any_sync(0xffffffffu, kmax < kKeys);
      // One pass over S computes P against the bound in use.  Its sum tells whether the bound
      // still holds (f16 takes P up to 65504): only where it does not, or before a row's first
      // key, is the row's maximum looked for, the bound moved and the pass repeated.
      uint32_t pk[kKeys / 2];
      float sum = 0.f, raw = 0.f;
      bool nan_row = false;
      auto scores = [&](uint32_t (&buf)[kKeys / 32][32]) {
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c) tmem_ld32_async(t_s + c * 32, buf[c]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c) tmem_ready32(buf[c]);
      };
      auto row_max = [&](float msub) {  // relative to msub
        uint32_t buf[kKeys / 32][32];
        scores(buf);
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < BL; ++b) {
          const float4 f = s_par[b];
          if (f.x != f.x) continue;
          float m = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (b * 16 + i < kmax)
              m = fmaxf(m, __uint_as_float(buf[b >> 1][(b & 1) * 16 + i]));
          mx = fmaxf(mx, fmaf(m, f.x, f.y - msub));
        }
        return mx;
      };
      auto pass = [&](auto masked, float msub) {
        uint32_t buf[kKeys / 32][32];
        scores(buf);
        float2 l2 = make_float2(0.f, 0.f), r2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int b = 0; b < BL; ++b) {
          const float4 f = s_par[b];
          float kf = f.x, nm = f.y - msub;
          if (kf != kf) {  // NaN for the rows that see the block, nothing for the others
            nan_row |= b * 16 < kmax;
            kf = 1.f;
            nm = -INFINITY;
          }
          float2 rs = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const int u = (b & 1) * 16 + i;
            float2 sv = make_float2(__uint_as_float(buf[b >> 1][u]),
                                    __uint_as_float(buf[b >> 1][u + 1]));
            if constexpr (decltype(masked)::value) {
              if (b * 16 + i >= kmax) sv.x = -INFINITY;
              if (b * 16 + i + 1 >= kmax) sv.y = -INFINITY;
            }
            const float2 xv = fma2(sv, make_float2(kf, kf), make_float2(nm, nm));
            const float2 pv = make_float2(ex2c(xv.x), ex2c(xv.y));
            rs = add2(rs, pv);
            pk[b * 8 + i / 2] = P8Io<__half>::pack(pv.x, pv.y);
          }
          r2 = add2(r2, rs);
          l2 = fma2(rs, make_float2(f.z, f.z), l2);
        }
        sum = l2.x + l2.y;
        raw = r2.x + r2.y;
      };
      bool move = m_used == -INFINITY && kmax > 0;
      for (int tries = 0; tries < 4; ++tries) {  // two are enough for finite scores
        if (__any_sync(0xffffffffu, move)) {
          const float mx = row_max(m_used == -INFINITY ? 0.f : m_used);
          const bool had = m_used != -INFINITY, grow = move && mx > (had ? 0.f : -INFINITY);
          const float alpha = grow && had ? ex2c(-mx) : 1.f;
          if (grow) m_used = (had ? m_used : 0.f) + mx;
          l *= alpha;
          if (__any_sync(0xffffffffu, grow && had)) {
            // O_x holds the earlier tiles' P V, once the last of them is done
            if (!wait_warp(&bars->o_full[x][(j - 1) & 1], ((j - 1) >> 1) & 1, abort_flag, p.err,
                           kErrTimeoutTmem, 78)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_ld16_async(t_o + c, o);
              tmem_wait16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(t_o + c, o);
            }
          }
        }
        const float msub = m_used == -INFINITY ? 0.f : m_used;
        if (edge) pass(std::true_type{}, msub);
        else pass(std::false_type{}, msub);
        move = raw > kMostSum;
        if (!__any_sync(0xffffffffu, move)) break;
      }
      if (!ok) break;
      l += nan_row ? __uint_as_float(0x7fc00000u) : sum;
#pragma unroll
      for (int c = 0; c < kKeys / 2; c += 16) tmem_st16(t_s + c, pk + c);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_full[x][j & 1]);
    }
    const int64_t orow = static_cast<int64_t>(row0 + tok) * p.Hq + h * p.G + r % p.G;
    if (n > 0) {
      if (ok && wait_warp(&bars->o_full[x][(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, p.err,
                          kErrTimeoutTmem, 90)) {
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tmem_ld32(t_o + c, o);
          tmem_wait_ld();
          if (!mine) continue;
          if (p.splits == 1) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + orow * D + c);
#pragma unroll
            for (int u = 0; u < 32; u += 8)
              dst[u / 8] = make_uint4(P8Io<T>::pack(o[u] * inv, o[u + 1] * inv),
                                      P8Io<T>::pack(o[u + 2] * inv, o[u + 3] * inv),
                                      P8Io<T>::pack(o[u + 4] * inv, o[u + 5] * inv),
                                      P8Io<T>::pack(o[u + 6] * inv, o[u + 7] * inv));
          } else {
            float4* dst =
                reinterpret_cast<float4*>(p.ws_o + (orow * p.splits + split) * D + c);
#pragma unroll
            for (int u = 0; u < 32; u += 4)
              dst[u / 4] = make_float4(o[u] * inv, o[u + 1] * inv, o[u + 2] * inv, o[u + 3] * inv);
          }
        }
      }
    } else if (mine && p.splits == 1) {  // no visible key
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + orow * D);
#pragma unroll
      for (int c = 0; c < D / 8; ++c) dst[c] = make_uint4(0, 0, 0, 0);
    }
    if (mine && p.lse != nullptr)
      p.lse[orow * p.splits + split] = l == 0.f ? -INFINITY : m_used + log2f(l);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == Cfg::MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM);
  }
}

// --------------------------------------------------------------------------- weights
struct MassParams {
  const int32_t* table;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  int max_pages, blocks;
  int64_t num_pages;
  const float4* par;
  const float* lse;            // [N * Hq]
  const float* mass_in;
  float* mass_out;
  int64_t N;
  int Hq, Hkv, G;
  int parts;                   // CTAs of a key tile's cluster
  int* err;
};

template <int D>
struct MassCfg {
  static constexpr int STAGES = 3;
  static constexpr int GROUPS = 4;             // of four warps; each has a score tile of its own
  static constexpr int CHUNKS = D / 64;
  static constexpr int TILE = kT * D * 2;
  static constexpr int SMEM = (1 + STAGES) * TILE + 1024 + 512 + GROUPS * kT * 12;
  static constexpr int PRODUCER = 4 * GROUPS, MMA = PRODUCER + 1;
  static constexpr int THREADS = (MMA + 1) * 32;
  static constexpr uint32_t TMEM = GROUPS * kT;
};

struct MassBars {
  uint64_t k_full;
  uint64_t q_full[3];
  uint64_t q_empty[3];
  uint64_t s_full[4];
  uint64_t s_empty[4];
  uint64_t mma_done;
  uint32_t tmem;
  int abort;
};

template <typename T, int D>
__global__ void __launch_bounds__(MassCfg<D>::THREADS, 1)
    p8_chunk_mass_kernel(const __grid_constant__ CUtensorMap tmQ,
                         const __grid_constant__ CUtensorMap tmK, const MassParams p) {
  using Cfg = MassCfg<D>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sK = smem;
  uint8_t* sQ = sK + Cfg::TILE;
  constexpr int GR = Cfg::GROUPS;
  float* s_lse = reinterpret_cast<float*>(sQ + STAGES * Cfg::TILE);  // [GR][128]
  int* s_lim = reinterpret_cast<int*>(s_lse + GR * kT);              // [GR][128]
  float* s_w = reinterpret_cast<float*>(s_lim + GR * kT);            // [GR][128]
  MassBars* bars = reinterpret_cast<MassBars*>(s_w + GR * kT);
  volatile int* abort_flag = &bars->abort;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int h = blockIdx.y, seq = blockIdx.z;
  const int part = static_cast<int>(cluster_ctarank());
  const int k0 = static_cast<int>(blockIdx.x) / p.parts * kT;
  const int row0 = __ldg(p.cu_q + seq), q_len = __ldg(p.cu_q + seq + 1) - row0;
  if (row0 < 0 || q_len < 0 || static_cast<int64_t>(row0) + q_len > p.N) {
    if (threadIdx.x == 0) report_error(p.err, kErrBounds, 91);
    p8_grid_wait();
    return;
  }
  const int kv = p8_len(p.kv_lens, seq, p.max_pages, p.err, 92);
  if (k0 >= kv) {
    p8_grid_wait();
    return;
  }
  const int start = kv - q_len, TT = kT / p.G;
  // this CTA's row tiles: part, part + parts, .. of those that see the keys
  const int i0 = max(0, k0 - start) / TT + part;
  const int n = max(0, ((q_len + TT - 1) / TT - i0 + p.parts - 1) / p.parts);
  const int64_t sh = static_cast<int64_t>(seq) * p.Hkv + h;

  if (threadIdx.x == 0) {
    mbar_init(&bars->k_full, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&bars->q_full[s], 1);
      mbar_init(&bars->q_empty[s], 1);
    }
    for (int x = 0; x < GR; ++x) {
      mbar_init(&bars->s_full[x], 1);
      mbar_init(&bars->s_empty[x], 4);
    }
    mbar_init(&bars->mma_done, 1);
    bars->abort = 0;
    fence_barrier_init();
  }
  {
    const int used = TT * p.G, rows = kT - used;
    for (int i = threadIdx.x; i < STAGES * Cfg::CHUNKS * rows * 8; i += blockDim.x) {
      const int t = i / (rows * 8), r = i % (rows * 8);
      *reinterpret_cast<uint4*>(sQ + t * (kT * 128) + used * 128 + r * 16) =
          make_uint4(0, 0, 0, 0);
    }
    if (rows > 0) fence_proxy_async_shared();
  }
  if (warp == Cfg::MMA) tmem_alloc(&bars->tmem, Cfg::TMEM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  p8_grid_wait();

  if (warp == Cfg::PRODUCER) {
    if (elect_one()) {
      mbar_arrive_expect_tx(&bars->k_full, Cfg::TILE);
#pragma unroll
      for (int c = 0; c < Cfg::CHUNKS; ++c)
        tma_load_4d(sK + c * kT * 128, &tmK, &bars->k_full, c * 64, k0, h, seq);
      int issued = 0;
      for (int i = 0; i < n; ++i) {
        const int st = i % STAGES;
        if (!mbar_wait(&bars->q_empty[st], ((i / STAGES) & 1) ^ 1, abort_flag, p.err,
                       kErrTimeoutEmpty, 93))
          break;
        mbar_arrive_expect_tx(&bars->q_full[st], Cfg::CHUNKS * TT * p.G * 128);
#pragma unroll
        for (int c = 0; c < Cfg::CHUNKS; ++c)
          tma_load_4d(sQ + st * Cfg::TILE + c * kT * 128, &tmQ, &bars->q_full[st], c * 64, 0, h,
                      row0 + (i0 + i * p.parts) * TT);
        ++issued;
      }
      drain(&bars->k_full, 0);
      for (int i = issued - STAGES < 0 ? 0 : issued - STAGES; i < issued; ++i)
        drain(&bars->q_full[i % STAGES], (i / STAGES) & 1);
    }
  } else if (warp == Cfg::MMA) {
    if (elect_one()) {
      constexpr uint32_t IDESC = idesc16<T>(kT, kT, false);
      bool ok = mbar_wait(&bars->k_full, 0, abort_flag, p.err, kErrTimeoutFull, 94);
      const uint32_t k_base = smem_u32(sK);
      for (int i = 0; i < n && ok; ++i) {
        const int st = i % STAGES, x = i % GR;
        if (!mbar_wait(&bars->q_full[st], (i / STAGES) & 1, abort_flag, p.err, kErrTimeoutFull,
                       95) ||
            !mbar_wait(&bars->s_empty[x], ((i / GR) & 1) ^ 1, abort_flag, p.err, kErrTimeoutTmem,
                       96)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t q_base = smem_u32(sQ + st * Cfg::TILE);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * (kT * 128) + (kk & 3) * 32;
          umma_bf16(tmem + x * 128, sw128_desc(k_base + off, 16, 1024),
                    sw128_desc(q_base + off, 16, 1024), IDESC, kk != 0 ? 1u : 0u);
        }
        umma_commit(&bars->s_full[x]);
        umma_commit(&bars->q_empty[st]);
      }
      umma_commit(&bars->mma_done);
      drain(&bars->mma_done, 0);
    }
  } else {
    const int x = warp >> 2, wq = warp & 3;
    const int r = wq * 32 + lane;                       // key of this thread; also its column
    const int key = k0 + r;
    const float kf = key < kv ? __ldg(&p.par[sh * p.blocks + key / kP8Page].x) : 0.f;
    const uint32_t t_s = tmem + x * 128 + (static_cast<uint32_t>(wq * 32) << 16);
    float2 acc[2] = {};
    bool ok = true;  // a warp that gave up still meets the others at their barriers
    // column r of a row tile: its log-sum-exp (one tile ahead) and last visible key
    const int my_tok = r / p.G;
    const float* my_lse =
        p.lse + static_cast<int64_t>(row0 + my_tok) * p.Hq + h * p.G + r % p.G;
    auto is_row = [&](int i) {
      return r < TT * p.G && (i0 + i * p.parts) * TT + my_tok < q_len;
    };
    auto fetch = [&](int i) {
      return i < n && is_row(i)
                 ? __ldg(my_lse + static_cast<int64_t>(i0 + i * p.parts) * TT * p.Hq)
                 : INFINITY;
    };
    float next = fetch(x);
    for (int i = x; i < n; i += GR) {
      const float le = next == -INFINITY ? INFINITY : next;  // a row without keys weighs nothing
      next = fetch(i + GR);
      named_bar_sync(1 + x, 128);                         // the previous tile's values are read
      s_lse[x * kT + r] = -le;
      s_lim[x * kT + r] = is_row(i) ? start + (i0 + i * p.parts) * TT + my_tok : -1;
      named_bar_sync(1 + x, 128);
      const int t0 = (i0 + i * p.parts) * TT;
      const bool edge = k0 + kT - 1 > start + t0 || t0 + TT > q_len;
      ok = ok && wait_warp(&bars->s_full[x], (i / GR) & 1, abort_flag, p.err, kErrTimeoutTmem, 97);
      if (!ok) continue;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kT; c += 32) {
        float s[32];
        tmem_ld32(t_s + c, s);
        tmem_wait_ld();
        if (c == kT - 32) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->s_empty[x]);
        }
#pragma unroll
        for (int u = 0; u < 32; u += 4) {
          const float4 nl = *reinterpret_cast<const float4*>(s_lse + x * kT + c + u);
          const float2 a = fma2(make_float2(s[u], s[u + 1]), make_float2(kf, kf),
                                make_float2(nl.x, nl.y));
          const float2 b = fma2(make_float2(s[u + 2], s[u + 3]), make_float2(kf, kf),
                                make_float2(nl.z, nl.w));
          float2 ea = make_float2(ex2c(a.x), ex2c(a.y)), eb = make_float2(ex2c(b.x), ex2c(b.y));
          if (edge) {
            const int4 li = *reinterpret_cast<const int4*>(s_lim + x * kT + c + u);
            if (key > li.x) ea.x = 0.f;
            if (key > li.y) ea.y = 0.f;
            if (key > li.z) eb.x = 0.f;
            if (key > li.w) eb.y = 0.f;
          }
          acc[0] = add2(acc[0], ea);
          acc[1] = add2(acc[1], eb);
        }
      }
    }
    const float w = (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
    s_w[x * kT + r] = w;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == Cfg::MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM);
  }
  __syncwarp();
  cluster_sync_all();  // every part's sums are in its shared memory
  if (part == 0 && threadIdx.x < kT && k0 + static_cast<int>(threadIdx.x) < kv) {
    const int key = k0 + threadIdx.x;
    float w = 0.f;
    for (int i = 0; i < p.parts; ++i)
#pragma unroll
      for (int x = 0; x < GR; ++x) {
        float y;
        asm volatile("ld.shared::cluster.f32 %0, [%1];"
                     : "=f"(y)
                     : "r"(mapa_shared(smem_u32(s_w + x * kT + threadIdx.x), i))
                     : "memory");
        w += y;
      }
    const int64_t page = p8_page(p.table + static_cast<int64_t>(seq) * p.max_pages, key / kP8Page,
                                 p.num_pages, p.err, 98);
    const int64_t at = (page * p.Hkv + h) * kP8Page + key % kP8Page;
    p.mass_out[at] = p.mass_in[at] + w;
  }
  __syncwarp();
  cluster_sync_all();  // nobody leaves while its sums are read
}

template <typename T, int FMT, int D>
int launch_expand(const P8Cache& c, const P8Seqs& s, const P8Attn& a, int blocks, int* err,
                  cudaStream_t st) {
  const int64_t units = static_cast<int64_t>(blocks) * c.Hkv * 2;
  if (units > 0x7fffffff) return -3;
  return p8_launch(p8_expand_kernel<T, FMT, D>,
                   dim3(static_cast<unsigned>((units + 7) / 8), s.num_seqs), 256, 0, st, c, s,
                   blocks, static_cast<unsigned>(units), a.scale * 1.4426950408889634f,
                   static_cast<T*>(a.ws_k), static_cast<__half*>(a.ws_v),
                   static_cast<float4*>(a.ws_par), err);
}

template <typename T, int D, int NQ>
int launch_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
               ChunkParams p, int max_q_len, int num_seqs, cudaStream_t st) {
  using Cfg = ChunkCfg<D, NQ>;
  constexpr auto kern = p8_chunk_kernel<T, D, NQ>;
  const int per_cta = NQ * (kT / p.G);
  p.row_ctas = (max_q_len + per_cta - 1) / per_cta;
  p.max_q_len = max_q_len;
  p.num_seqs = num_seqs;
  const int64_t gx = static_cast<int64_t>(p.row_ctas) * p.splits * p.Hkv * num_seqs;
  if (gx > 0x7fffffff) return -3;
  const int rc = p8_opt_in<kern>(Cfg::SMEM);
  if (rc) return rc;
  return p8_launch(kern, dim3(static_cast<unsigned>(gx)), Cfg::THREADS, Cfg::SMEM, st, tq, tk, tv, p);
}

template <typename T, int D>
int launch_chunk(const P8Cache& c, const P8Seqs& s, const P8Attn& a, int* err, cudaStream_t st) {
  const int blocks = p8_chunk_blocks(s);
  int rc = c.fmt == kP8Int8 ? launch_expand<T, kP8Int8, D>(c, s, a, blocks, err, st)
                            : launch_expand<T, kP8E4m3, D>(c, s, a, blocks, err, st);
  if (rc) return rc;
  const int G = a.Hq / c.Hkv, TT = kT / G;
  CUtensorMap tq, tk, tv;
  {
    const int64_t dims[4] = {D, G, c.Hkv, a.N};
    const int64_t strides[3] = {D * 2, static_cast<int64_t>(G) * D * 2, a.q_stride * 2};
    const int box[4] = {64, G, 1, TT};
    rc = make_tmap_nd(&tq, a.q, 4, dims, strides, box, false, true);
  }
  const int64_t Lw = static_cast<int64_t>(blocks) * kP8Page;
  Bhsd k, v;
  k.p = a.ws_k;
  v.p = a.ws_v;
  k.ss = v.ss = D;
  k.sh = v.sh = Lw * D;
  k.sb = v.sb = Lw * D * c.Hkv;
  if (!rc) rc = make_bhsd_map(&tk, k, s.num_seqs, c.Hkv, static_cast<int>(Lw), D, kKeys);
  if (!rc) rc = make_bhsd_map(&tv, v, s.num_seqs, c.Hkv, static_cast<int>(Lw), D, kKeys);
  if (rc) return rc;
  ChunkParams p;
  p.cu_q = s.cu_q;
  p.kv_lens = s.kv_lens;
  p.max_pages = s.max_pages;
  p.blocks = blocks;
  p.par = static_cast<const float4*>(a.ws_par);
  p.out = a.out;
  p.lse = a.ws_lse;
  p.ws_o = a.ws_o;
  p.N = a.N;
  p.Hq = a.Hq;
  p.Hkv = c.Hkv;
  p.G = G;
  p.splits = a.splits;
  p.row_ctas = p.max_q_len = 0;  // set at the launch
  p.err = err;
  const bool mass = a.mass_out != nullptr;
  rc = a.chunk_nq == 2 ? launch_fwd<T, D, 2>(tq, tk, tv, p, a.max_q_len, s.num_seqs, st)
                       : launch_fwd<T, D, 1>(tq, tk, tv, p, a.max_q_len, s.num_seqs, st);
  if (rc) return rc;
  if (p.splits > 1) {
    rc = p8_combine(s, a, c.D, st);
    if (rc) return rc;
  }
  if (mass) {
    using Cfg = MassCfg<D>;
    CUtensorMap tkm;
    rc = make_bhsd_map(&tkm, k, s.num_seqs, c.Hkv, static_cast<int>(Lw), D, kT);
    if (rc) return rc;
    MassParams m;
    m.table = s.table;
    m.cu_q = s.cu_q;
    m.kv_lens = s.kv_lens;
    m.max_pages = s.max_pages;
    m.blocks = blocks;
    m.num_pages = c.num_pages;
    m.par = p.par;
    m.lse = p.splits > 1 ? a.ws_total : a.ws_lse;
    m.mass_in = a.mass_in;
    m.mass_out = a.mass_out;
    m.N = a.N;
    m.Hq = a.Hq;
    m.Hkv = c.Hkv;
    m.G = G;
    m.err = err;
    constexpr auto kern = p8_chunk_mass_kernel<T, D>;
    rc = p8_opt_in<kern>(Cfg::SMEM);
    if (rc) return rc;
    const int key_tiles = (s.max_pages * kP8Page + kT - 1) / kT;
    const int64_t ctas = static_cast<int64_t>(key_tiles) * c.Hkv * s.num_seqs;
    const int row_tiles = (a.max_q_len + TT - 1) / TT;
    m.parts = 1;
    while (m.parts < 8 && 2 * m.parts * ctas <= a.num_sms && 8 * m.parts <= row_tiles)
      m.parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = m.parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cfg.stream = st;
    cfg.gridDim = dim3(key_tiles * m.parts, c.Hkv, s.num_seqs);
    cfg.blockDim = dim3(Cfg::THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tq, tkm, m);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

// Both paths at 64 rows, D 128: 16 requests of 2048 tokens 76 us (paged8_attn.cu) and 63 us (here),
// one of 2048 16.4 and 17.0,
// one of 32768 72.2 and 71.4, 8 of 16384 187 and 231; at 32 rows 16 of 2048 take 42 and 61.
bool p8_is_chunk(int max_q_len, int group) {
  return static_cast<int64_t>(max_q_len) * group > kP8ShortRows;
}

void p8_chunk_plan(const P8Seqs& s, int Hkv, int group, int max_q_len, int num_sms, int* nq,
                   int* splits) {
  const int TT = kT / group;
  const int64_t heads = static_cast<int64_t>(Hkv) * s.num_seqs;
  const int64_t pairs = (max_q_len + 2 * TT - 1) / (2 * TT) * heads;
  // two row tiles share the keys of a CTA once that still fills the SMs
  *nq = pairs >= num_sms ? 2 : 1;
  // one row tile a CTA: two CTAs on an SM, at least eight key tiles each
  const int64_t ctas = (max_q_len + TT - 1) / TT * heads;
  const int64_t tiles = (static_cast<int64_t>(s.max_pages) * kP8Page + kKeys - 1) / kKeys;
  int64_t sp = *nq == 2 ? 1 : 2 * num_sms / ctas;
  if (sp > tiles / 8) sp = tiles / 8;
  *splits = static_cast<int>(sp < 1 ? 1 : sp);
}

int p8_chunk_blocks(const P8Seqs& s) {
  constexpr int per = kT / kP8Page;
  return (s.max_pages + per - 1) / per * per;
}

int p8_chunk_attention(const P8Cache& c, const P8Seqs& s, const P8Attn& a, int* err,
                       cudaStream_t stream) {
  if (a.N <= 0 || s.num_seqs <= 0) return 0;
  if (s.num_seqs > 65535 || c.Hkv > 65535 || a.Hq / c.Hkv > kT) return -3;
  if (a.type == kP8Bf16)
    return c.D == 128 ? launch_chunk<__nv_bfloat16, 128>(c, s, a, err, stream)
                      : launch_chunk<__nv_bfloat16, 64>(c, s, a, err, stream);
  return c.D == 128 ? launch_chunk<__half, 128>(c, s, a, err, stream)
                    : launch_chunk<__half, 64>(c, s, a, err, stream);
}

}  // namespace cfb
