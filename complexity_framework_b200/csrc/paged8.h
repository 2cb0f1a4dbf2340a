// Host launchers of the 8-bit paged KV cache kernels (paged8_cache.cu, paged8_attn.cu).
//
// One layer of the cache:
//   codes  [pages, Hkv, 2, 16, D]  int8 or e4m3; K then V of a (page, head) are contiguous
//   scales [pages, Hkv, 2]         fp32, one for each block of 16 tokens, head and K / V
//   mass   [pages, Hkv, 16]        fp32, accumulated attention weight (optional)
// page_table [S, max_pages], cu_q [S + 1], kv_lens [S] are int32.  Sequence i owns the
// rows [cu_q[i], cu_q[i+1]) of the new tokens, which sit at the last positions of its
// kv_lens[i] cached tokens; a row whose position is negative has no token and no output.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace cfb {

constexpr int kP8Page = 16;  // tokens of a page, and of a scale block
// Rows (new tokens x query heads of a KV head) up to which a chunk takes the decode kernel.
constexpr int kP8ShortRows = 64;

enum P8Fmt : int { kP8Int8 = 0, kP8E4m3 = 1 };
enum P8Type : int { kP8Bf16 = 0, kP8Half = 1 };

struct P8Cache {
  uint8_t* codes = nullptr;
  float* scales = nullptr;
  int64_t num_pages = 0;
  int Hkv = 0, D = 0, fmt = kP8Int8;
};

struct P8Seqs {
  const int32_t* table = nullptr;
  const int32_t* cu_q = nullptr;
  const int32_t* kv_lens = nullptr;
  int num_seqs = 0, max_pages = 0;
};

// Quantises the new tokens' k, v [N, Hkv, D] (row strides in elements) into their blocks.
// Their mass (where there is one) becomes 0.
int p8_append(const P8Cache& c, const P8Seqs& s, const void* k, int64_t k_stride, const void* v,
              int64_t v_stride, int64_t N, int max_q_len, int type, float* mass, int* err,
              cudaStream_t stream);

// k_out, v_out [layers, S, Hkv, max_pages * 16, D]: the cached values, 0 past kv_lens.
int p8_read(const P8Cache& c, const P8Seqs& s, int layers, void* k_out, void* v_out, int type,
            int* err, cudaStream_t stream);

struct P8Attn {
  const void* q = nullptr;   // [N, Hq, D], row stride q_stride elements
  int64_t q_stride = 0;
  void* out = nullptr;       // [N, Hq, D]
  int type = kP8Bf16;
  int64_t N = 0;
  int Hq = 0, max_q_len = 1;
  float scale = 1.f;
  const float* mass_in = nullptr;  // with mass_out: mass_out = mass_in + weights
  float* mass_out = nullptr;
  // long chunks only
  int splits = 1;
  float* ws_o = nullptr;     // [N * Hq, splits, D] (splits > 1)
  float* ws_lse = nullptr;   // [N * Hq, splits] (splits > 1 or mass)
  float* ws_total = nullptr; // [N * Hq] (splits > 1 and mass)
  int chunk_nq = 2;          // 128-row tiles of a CTA
  int num_sms = 148;
  // keys and values as 16-bit operands, Lw = 16 * p8_chunk_blocks() tokens
  void* ws_k = nullptr;      // [S, Hkv, Lw, D]
  void* ws_v = nullptr;
  void* ws_par = nullptr;    // float4 [S, Hkv, Lw / 16]
};

// Decode and short chunks: how the work is dealt out, and the workspace in floats.
struct P8AttnPlan {
  int nb = 1;                // 8-row tiles of a CTA
  int row_tiles = 1;         // row tiles of the longest chunk
  int chunk = 1, splits = 1; // pages of a CTA, CTAs of the longest (sequence, KV head, row tile)
  int score_rows = 4;        // rows of a token's kept scores (mass)
  int64_t n_o = 0, n_lse = 0, n_s = 0;
  int64_t floats() const { return n_o + n_lse + n_s; }
};
P8AttnPlan p8_attn_plan(const P8Cache& c, const P8Seqs& s, int group, int max_q_len, bool mass,
                        int num_sms);
int p8_attention(const P8Cache& c, const P8Seqs& s, const P8Attn& a, const P8AttnPlan& plan,
                 float* ws, int* err, cudaStream_t stream);

// Long chunks.  Joins the splits of the sequences' rows: out, and each row's total, from ws_o
// and ws_lse.
int p8_combine(const P8Seqs& s, const P8Attn& a, int D, cudaStream_t stream);
int p8_chunk_blocks(const P8Seqs& s);
// Whether a call's chunks go to the tcgen05 kernels.
bool p8_is_chunk(int max_q_len, int group);
// Row tiles of a CTA and KV splits of the chunk kernel.
void p8_chunk_plan(const P8Seqs& s, int Hkv, int group, int max_q_len, int num_sms, int* nq,
                   int* splits);
int p8_chunk_attention(const P8Cache& c, const P8Seqs& s, const P8Attn& a, int* err,
                       cudaStream_t stream);

// Keeps `budget` tokens of each sequence and moves them to the pages of dst_table
// [S, dst_pages]; keep [layers, S, Hkv, budget] int32.
int p8_evict(const P8Cache& c, const P8Seqs& s, float* mass, int layers, const int32_t* dst_table,
             int dst_pages, int budget, int recent, int32_t* keep, int* err, cudaStream_t stream);

}  // namespace cfb
