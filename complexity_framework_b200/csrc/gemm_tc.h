// Host interface of the tcgen05 GEMM (see gemm_tc.cu for the kernel design).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace cfb {

enum GemmEpilogue : int {
  EPI_STORE = 0,       // C(bf16) = alpha * acc
  EPI_RESID = 1,       // C(bf16) = alpha * acc + R(bf16)
  EPI_SWIGLU_FWD = 2,  // gate|up tile -> GU(bf16 pre-activations), ACT = silu(g)*u*scale
  EPI_SWIGLU_BWD = 3,  // acc = d(ACT) -> C = d(GU) using saved GU
  EPI_F32 = 4,         // C(fp32) = alpha * acc
  EPI_F32_ACC = 5,     // C(fp32) += alpha * acc
  EPI_F32_ATOMIC = 7,  // C(fp32) += alpha * acc with atomics; K may be split across CTAs
  EPI_CE_STATS = 6,    // C(bf16) logits = alpha*acc; stats[row, N/128] = (max, sumexp); BN=256
  EPI_PEER_STORE = 8,  // reduce-scatter partials: owner = row / peer_rows; fp32 tile stored
                       // over NVLink into peer_c[owner][sync.rank][row % peer_rows][col]
  EPI_CE_FWD = 9,      // nothing of C is stored: per (row, 128 columns) softmax statistics and
                       // the target's logit; BN=256 (see GemmCe)
  EPI_CE_GRAD = 10,    // C(bf16) = d(loss)/d(logits) of the columns' part of the vocabulary
};

constexpr int kMaxSeg = 8;

// Device barrier over symmetric-memory signal pads (int[rounds][kMaxSeg] per
// rank).  `role` 1: the TMA producer waits before its first load (operands
// that live in peer memory must be written); role 2: the epilogue waits
// before its first peer store (peer destinations must be cleared).  With
// `signal`, CTA 0 first announces this rank's arrival.  world == 0: none.
struct DistSync {
  int* pad[kMaxSeg] = {};
  int world = 0;
  int rank = 0;
  int round = 0;
  int epoch = 0;
  int role = 0;
  int signal = 0;
};

// Width (in activation columns) of one gate block in the packed gate|up weight:
// packed rows [256j, 256j+128) are gate rows [128j, 128j+128) and rows
// [256j+128, 256j+256) the matching up rows.
constexpr int kSwigluBlock = 128;

// All-gather of A's row shards performed inside the GEMM: warp 2 of every CTA
// copies 128-row chunks of the peers' shards (P2P loads) into this rank's
// gathered buffer `dst` (the A operand) and publishes a per-chunk flag; the
// TMA producer waits for a chunk's flag before loading its rows.  Tiles of
// this rank's own rows are scheduled first.  src[q] is rank q's gathered
// buffer, whose rows [q*rows, (q+1)*rows) hold q's shard.
struct AgCopy {
  const __nv_bfloat16* src[kMaxSeg] = {};
  __nv_bfloat16* dst = nullptr;
  int* flags = nullptr;  // one per 128-row chunk of dst
  int rows = 0;          // rows per rank
  int cols = 0;          // row length (elements) of src/dst
  int epoch = 0;
  int active = 0;
};

// Grouped GEMMs (expert-parallel work inside one launch).
//  mode 1, row-grouped: the A rows are sorted into per-group segments padded to
//    the 256-row tile; tile_group[m_tile] is the group of each 256-row tile (< 0:
//    no work) and B's storage rows of group g start at g * b_stride (N rows of a
//    K-major B, K rows of an MN-major B).
//  mode 2, K-grouped (weight gradients): group g multiplies the K rows
//    [k_start[g], k_start[g+1]) of MN-major A and B (multiples of 64) into output
//    rows [g * c_stride, g * c_stride + M); work units are (group, tile, K slice).
// The tables live in device memory, so segment sizes never reach the host.
struct GemmGroups {
  int mode = 0;
  const int* tile_group = nullptr;
  const int* k_start = nullptr;
  int ngroups = 0;
  int64_t b_stride = 0;
  int64_t c_stride = 0;
};

// Cross-entropy epilogues: acc is h . w of a row and a word, its logit z = scale * acc and
// t = k2 * acc the same in units of log 2.
struct GemmCe {
  float k2 = 0.f;     // scale * log2(e)
  float scale = 1.f;  // logit scale
  const int* target = nullptr;  // [M] word of each row, < 0: none
  // forward: (m, sum 2^(k2 (acc - m))) of a half tile with m its largest acc, acc of the
  // target, and (where wanted) the sum of scale * acc over a half tile; scale > 0
  float2* stats = nullptr;  // [M][2 * ceil(N / 256)]
  float* zt = nullptr;      // [M]
  float* zsum = nullptr;    // [M][2 * ceil(N / 256)]
  // gradient: g_t (p (1 + 2 lambda lse) - eps / V - (1 - eps) [target]) / unit, where g_t is the
  // row's own factor (per_row) or 1, and unit is 1 - eps (1 where that is 0): the target's term of
  // a row without a factor is then -1, which bf16 holds exactly
  const float* lse2 = nullptr;  // [M] log-sum-exp in units of log 2
  const float* gout = nullptr;  // null, or one factor for each row of the call's own order
  const int* src = nullptr;     // [M] that order's row of each row here, < 0: none
  float inv_unit = 1.f;
  float z2 = 0.f;        // 2 lambda
  float smooth = 0.f;    // eps
  float smooth_v = 0.f;  // eps / V
  float* resid = nullptr;  // [M] the target's gradient less its rounded value
  int col0 = 0;          // first word of this call's columns
  int n_valid = 0;       // columns that are words (the others pad N to 32)
};

struct GemmEpi {
  void* c = nullptr;
  int64_t ldc = 0;
  const __nv_bfloat16* r = nullptr;
  int64_t ldr = 0;
  float alpha = 1.0f;
  __nv_bfloat16* gu = nullptr;
  int64_t ldgu = 0;
  __nv_bfloat16* act = nullptr;
  int64_t ldact = 0;
  const float* row_scale = nullptr;  // [M, n_experts]
  int shared_width = 0;
  int expert_width = 1;
  int n_experts = 0;
  float shared_scale = 1.0f;
  float* stats = nullptr;  // [M, 2*ceil(N/BN)] float2 (one per 128-column half tile)
  float* peer_c[kMaxSeg] = {};  // EPI_PEER_STORE: every rank's [world][peer_rows][ldc] fp32 slots
  int64_t peer_rows = 0;        // rows owned by each rank
  DistSync sync;
  AgCopy ag;
  GemmGroups grp;
  GemmCe ce;
  // sizes that the host does not know: fewer rows of C (m_dev) or of K (k_dev) than M or K
  const int* m_dev = nullptr;
  int m_off = 0;             // rows of m_dev before this launch's first
  const int* k_dev = nullptr;
  int64_t split_stride = 0;  // EPI_F32 / EPI_F32_ACC: K slices write their own C, this far apart
  const float* alpha_dev = nullptr;  // EPI_STORE, EPI_F32, EPI_F32_ACC: a further factor of acc
  int dependent = 0;         // launch before the end of the kernel before, and wait for it inside
  int group_m = 0;           // > 0: the schedule takes the row tiles in groups of this many, every
                             // column tile of a group before the next group
};

struct GemmArgs {
  const void* A = nullptr;
  int64_t lda = 0;
  bool a_mn = false;
  const void* B = nullptr;
  int64_t ldb = 0;
  bool b_mn = false;
  int M = 0, N = 0, K = 0;
  int epi = EPI_STORE;
  int bn = 0;  // 0 = choose
  int num_sms = 148;
  int n_valid = 0;  // > 0: B and C have this many columns only; N is it rounded up to 32
  int ksplit = 1;   // EPI_F32 / EPI_F32_ACC: K slices (at most one a 64-wide K block)
  // Operand segments (all-gather fused into the GEMM): when a_nseg > 0 the A
  // matrix is the concatenation, along its storage rows (M for K-major, K for
  // MN-major), of a_nseg matrices of a_seg_rows rows each, at A_seg[i] (peer
  // memory allowed; loads are plain TMA, never multicast).  Same for B.
  const void* A_seg[kMaxSeg] = {};
  int a_nseg = 0;
  int64_t a_seg_rows = 0;
  const void* B_seg[kMaxSeg] = {};
  int b_nseg = 0;
  int64_t b_seg_rows = 0;
};

int gemm_tc_launch(const GemmArgs& g, const GemmEpi& ep, cudaStream_t stream, int* err);
int choose_bn(int M, int N, int num_sms);
int make_tmap_2d(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld,
                 int box_inner, int box_outer);
// Tiled map of `rank` (<= 5) dims given innermost first; byte_strides[i] is the
// stride of dim i+1.  bf16 or fp32 elements, 128-byte swizzle or none.
int make_tmap_nd(CUtensorMap* map, const void* base, int rank, const int64_t* dims,
                 const int64_t* byte_strides, const int* box, bool fp32, bool swizzle128);
// 2-D map for epilogue stores: 32 x 32 boxes with 64-byte swizzle.
int make_tmap_2d_store(CUtensorMap* map, const void* base, int64_t rows, int64_t cols,
                       int64_t ld);

}  // namespace cfb
