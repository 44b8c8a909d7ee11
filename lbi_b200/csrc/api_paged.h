// C entry points of the serving operators over a paged key / value cache (paged_kv.cu, paged_attn.cu, logits.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { LBI_F32 = 0, LBI_BF16 = 1, LBI_F16 = 2, LBI_E4M3 = 3 };

// The cache and the batch that every operator reads.
//   k, v      [num_pages, kv_heads, page_size, head_dim], page_size a power of two in 8 .. 128
//   k_scale, v_scale  fp32 [num_pages, kv_heads, page_size], null unless cache_type is LBI_E4M3 (value = code * scale)
//   table     int32 [batch, table_width] (rows table_stride apart): page of every page_size positions of a sequence
//   context   int32 [batch]: tokens of the sequence, its new ones included
//   cu        int32 [batch + 1] row offsets of the sequences' new tokens, or null: rows / batch tokens each
typedef struct {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  const int* table;
  const int* context;
  const int* cu;
  int64_t table_stride;
  int num_pages, kv_heads, page_size, head_dim, cache_type;
  int table_width, batch;
  int rows;     // new tokens (rows of qkv / q); rows in front of the first sequence and behind the last belong to nobody
  int* status;  // device int: 83 a position outside the rotary table, 84 a position or page outside the page table or the pool
} lbi_paged_batch;

// qkv [rows, (heads + 2 kv_heads) * head_dim] (rows qkv_stride elements apart, type `type`): rotates q and k by the rotary table
// rows of their positions (cos / sin fp32 [rope_rows, head_dim / 2]; null: no turn), writes q_out [rows, heads * head_dim] and the
// k / v rows into their pages.  Rows in front of the first sequence and behind the last: q_out is left as it is, or zeroed when
// zero_tail is set.
int lbi_kv_append(const lbi_paged_batch* p, const void* qkv, int64_t qkv_stride, void* q_out, int type, int heads, const float* cos_tab,
                  const float* sin_tab, int64_t rope_rows, int interleaved, int zero_tail, cudaStream_t stream);

// k_out, v_out [batch, kv_heads, max_len, head_dim] of `type`: positions below the context length, zeros behind it.
int lbi_kv_gather(const lbi_paged_batch* p, void* k_out, void* v_out, int64_t max_len, int type, cudaStream_t stream);

// How a long context is cut: `splits` parts of `split_keys` keys (the last takes what is left).  With more than one part the caller
// supplies part_o fp32 [rows * heads, splits, head_dim] and part_lse fp32 [rows * heads, splits].
typedef struct {
  int kernel;   // 0 tiles of 16 rows for any type and head size, 1 tiles of 8 or 16 rows, 2 tiles of 256 rows
  int rows;     // of a tile of kernels 0 and 1
  int splits, split_keys;
} lbi_attention_plan;
lbi_attention_plan lbi_paged_attention_plan(const lbi_paged_batch* p, int type, int heads, float scale, int64_t max_context, int sm_count);

// out [rows, heads * head_dim] = causal attention of the new tokens q (row stride q_stride elements) over the sequences' pages.
int lbi_paged_attention(const lbi_paged_batch* p, const void* q, int64_t q_stride, void* out, float* part_o, float* part_lse,
                        lbi_attention_plan plan, int type, int heads, float scale, int zero_tail, int sm_count, cudaStream_t stream);

// out fp32 [batch, vocab] from logits [batch, vocab] (row stride, type), the rules of logits.cu.  Null pointers: the scalar is used.
typedef struct {
  const void* logits;
  int64_t logits_stride;
  float* out;
  int64_t out_stride;
  const int64_t* tokens;
  int64_t tokens_stride;
  const int* lengths;
  const int* prompt_lengths;
  const float* repetition_row;
  const float* presence_row;
  const float* frequency_row;
  const float* bias;
  int64_t bias_stride;   // 0: one row for the whole batch
  const int* allowed;
  int64_t allowed_stride;
  float repetition, presence, frequency;
  int type, batch, vocab, history;
} lbi_logit_rules;
int lbi_adjust_logits(const lbi_logit_rules* p, int sm_count, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
