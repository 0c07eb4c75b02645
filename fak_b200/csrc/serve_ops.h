// Launchers of the 4-bit KV cache, batch plan and log-probability kernels (plain pointers; the checks
// and the torch types are in serve_ops.cpp).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace fak {

enum class Elt : int { F32 = 0, F16 = 1, BF16 = 2 };

constexpr int kKv4LoadBytes = 16;   // what one vector load of the append takes of a row

struct Kv4Rows {   // k / v rows: element (token, head, d) at ptr + (tok / 16) * s_page + (tok % 16) * s_row + head * s_head + d
  const void* k;
  const void* v;
  int64_t ks_page, ks_row, ks_head, vs_page, vs_row, vs_head;
  Elt type;
  bool vec;   // every row of every page and head starts on kKv4LoadBytes
};
void kv4_append_launch(const Kv4Rows& r, const int* slot, int T, int Hkv, int D, uint8_t* pages, int64_t n_pages,
                       int* err, cudaStream_t stream);
void kv4_read_launch(const uint8_t* pages, int64_t n_pages, const int* slot, int T, int Hkv, int D, void* k, void* v,
                     Elt type, int* err, cudaStream_t stream);

struct Kv4Attn {
  const void* q;             // [T, H, D], row strides q_tok, q_head (elements)
  int64_t q_tok, q_head;
  Elt q_type;
  bool q_vec;                // rows start on 16 bytes
  const uint8_t* pages;      // [n_pages, Hkv, 20 D]
  int64_t n_pages;
  const int* table;          // [B, >= width]
  int64_t table_stride;
  int width;
  const int* q_off;          // [B + 1] or null: one query per sequence
  const int* ctx;            // [B]
  int n_tokens;              // rows of q
  int B, H, Hkv, D, max_new;
  int G;                     // query heads per KV head; row r of a (sequence, KV head) is query r / G, head r % G
  uint32_t g_inv;            // ceil(2^32 / G) for G > 1: r / G = (r g_inv) / 2^32 while r G < 2^32
  void* out;                 // [T, H, D], row strides o_tok, o_head
  int64_t o_tok, o_head;
  Elt o_type;
  bool o_vec;                // 16-bit rows that start on 16 bytes
  float scale, softcap;
  int window;
  const float* sinks;        // [H] or null
  int n_split;               // 0: chosen by the rule in kv4_attn.cu
  int tiles;                 // kernel: -1 by the rows, 0 warps over pages, 1 tiles of query rows
#ifdef __CUDACC__
  __device__ __forceinline__ int query_of(int r) const { return G == 1 ? r : (int)__umulhi((uint32_t)r, g_inv); }
#endif
  float* part;               // split partials (kv4_attn_plan)
  int* err;
};
struct Kv4AttnPlan {
  bool tc, cluster;   // tiles of query rows on tcgen05; the splits merge inside thread-block clusters
  int nt, row_chunks, n_split;
  int64_t whole;      // row blocks (of B * Hkv * row_chunks, in block_no's order) whose keys are not split
  int64_t part_floats;
};
Kv4AttnPlan kv4_attn_plan(const Kv4Attn& a, int n_sm);
void kv4_prefill_launch(const Kv4Attn& a, const Kv4AttnPlan& p, cudaStream_t stream);
void kv4_attn_launch(const Kv4Attn& a, const Kv4AttnPlan& p, cudaStream_t stream);

struct BatchPlanArgs {
  const int *old_len, *new_len;
  int B;
  int* table;
  int64_t table_stride;
  int width;
  const int* free_pages;
  int n_free;
  const int* head;
  int max_tokens;
  int *slot, *pos, *seq, *q_off, *ctx, *last, *head_out;
  int* err;
};
void batch_plan_launch(const BatchPlanArgs& a, cudaStream_t stream);

struct LogprobArgs {
  const void* x;
  Elt type;
  int64_t stride;
  int T, V, k;
  const int* target;
  float softcap;
  float *logprob, *entropy;
  int* rank;
  int* top_ids;
  float* top_logprobs;
  int n_seg;
  float* part;      // logprob_part_words(T, n_seg) when n_seg > 1: a record a segment
  int* tickets;     // [T] zeroed
  bool vec;
};
int logprob_segments(int T, int V, int n_sm);
int64_t logprob_part_words(int T, int n_seg);
void logprob_launch(const LogprobArgs& a, cudaStream_t stream);

}  // namespace fak
