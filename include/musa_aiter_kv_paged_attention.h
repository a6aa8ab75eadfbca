/*
 * C-ABI of libmusa_aiter_kv_hip.so, third part: operators on paged caches of plain values [blocks, kv_heads, head_dim,
 * block_size] -- attention with a sliding window and first tokens that stay visible, attention for trees of drafted
 * tokens, the attention weight that cached tokens gather, and the eviction of the tokens that gathered least.
 * None of them has a reference counterpart.
 *
 * As in musa_aiter_kv_serving.h every entry launches asynchronously on `stream` and returns the HIP status; nothing is
 * launched for arguments that are refused.  Tables, lengths, rows, masks and reference counts are read on the device
 * only, and every id read from them is checked there before it is used as an address.
 */
#ifndef MUSA_AITER_KV_PAGED_ATTENTION_H_
#define MUSA_AITER_KV_PAGED_ATTENTION_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Attention, and the weight that tokens gather ------------------------------------------------
 * query [rows, heads, head_dim] and caches [num_blocks, kv_heads, head_dim, block_size] of one type (dtype 0 f32,
 * 1 f16, 2 bf16; a block's values packed), tables [batch, max_blocks], lens [batch], starts [batch + 1] or NULL
 * (rows == batch, one row each); wide flags: 1 int64, 0 int32.
 *
 * masks NULL: row i of the n of a sequence of `len` cached tokens sits at pos = len - n + i and sees the positions up
 * to there; with window > 0 only those past pos - window and those below sinks.
 * masks [rows, mask_words]: the rows are the sequence's last n tokens, a tree of drafts.  Each sees the len - n
 * positions in front, and of the drafted token k < 64 * mask_words bit k % 64 of word k / 64 says whether it is seen
 * (window and sinks are 0 then).
 * Positions whose table entry is missing or outside the cache are not seen.
 *
 * musa_aiter_hip_paged_attention: out (packed, of query's type) and lse float32 [rows, heads] (or NULL).  A row that
 * sees nothing gives 0 and lse -inf.  Rows of no sequence are zeroed in out with fill_rows, else left as they are
 * there; their lse is -inf.  out and lse share no memory with what the call reads.  `longest` is an upper bound of
 * lens; only how the work is cut depends on it.  workspace holds musa_aiter_hip_paged_attention_workspace bytes (NULL
 * where that is 0).
 *
 * musa_aiter_hip_attention_weights (masks NULL; cache[1], out and the workspace are not used): adds to
 * weights[b, kv head, j] the sum of e^(score - lse) over the rows and heads of the kv head that see position
 * j < weight_tokens.  Rows whose lse is -inf give nothing.  The strides of weights are in elements. */
typedef struct musa_aiter_hip_paged_attention_call {
  const void* query;
  void* out;
  float* lse;
  const void* cache[2];
  const void* tables;
  const void* lens;
  const void* starts;
  const int64_t* masks;
  float* weights;
  void* workspace;
  int64_t workspace_bytes;
  int64_t rows, batch, heads, kv_heads, head_dim, block_size, num_blocks, max_blocks;
  int64_t query_row_stride, query_head_stride;              /* elements */
  int64_t cache_block_stride[2];                             /* bytes */
  int64_t table_stride;                                      /* elements between rows of tables */
  int64_t mask_words, mask_stride;                           /* words of a row, and between rows */
  int64_t window, sinks;
  int64_t longest;
  int64_t weight_tokens, weight_row_stride, weight_head_stride;
  double softmax_scale;
  int32_t dtype;
  int32_t wide_tables, wide_lens, wide_starts;
  int32_t fill_rows;
  int32_t reserved;
} musa_aiter_hip_paged_attention_call;
int musa_aiter_hip_paged_attention(const musa_aiter_hip_paged_attention_call* call, void* stream);
int64_t musa_aiter_hip_paged_attention_workspace(const musa_aiter_hip_paged_attention_call* call);
int musa_aiter_hip_attention_weights(const musa_aiter_hip_paged_attention_call* call, void* stream);

/* ---- Eviction ------------------------------------------------------------------------------------
 * The two caches share no memory (their blocks may lie between each other).
 * cache [layers, num_blocks, kv_heads, head_dim, block_size] of 1-, 2- or 4-byte elements (a block's packed, strides in
 * bytes), weights float32 [layers, batch, kv_heads, weight_tokens] (strides in elements, the last extent packed),
 * tables [batch, max_blocks], lens and keep [batch], refs [num_blocks] or NULL.
 * Row b keeps k = keep[b] of its lens[b] tokens, in every layer and kv head: the first min(sinks, k), the last
 * min(recent, what is left of k) and of those between the heaviest (equal weights: the earliest; a NaN is lighter than
 * any number, a position past weight_tokens weighs 0).  They move in order to the positions [0, k), their weights with
 * them, and the weights of [k, len) become 0; the cache past k stays as it is.  kept[b] = k.
 * A row is left as it is, kept[b] = max(lens[b], 0), where keep[b] is negative or not below lens[b], where one of its
 * pages is missing or outside the cache, and where refs counts more than one owner of one of them. */
typedef struct musa_aiter_hip_evict_call {
  void* cache[2];
  float* weights;
  const void* tables;
  const void* lens;
  const void* keep;
  const void* refs;
  int64_t* kept;
  void* workspace;
  int64_t workspace_bytes;
  int64_t layers, batch, kv_heads, head_dim, block_size, num_blocks, max_blocks, element_bytes;
  int64_t cache_layer_stride[2], cache_block_stride[2];     /* bytes */
  int64_t weight_tokens, weight_layer_stride, weight_row_stride, weight_head_stride;
  int64_t table_stride;
  int64_t sinks, recent;
  int32_t wide_tables, wide_lens, wide_keep, wide_refs;
} musa_aiter_hip_evict_call;
int musa_aiter_hip_evict(const musa_aiter_hip_evict_call* call, void* stream);
int64_t musa_aiter_hip_evict_workspace(const musa_aiter_hip_evict_call* call);

#ifdef __cplusplus
}
#endif

#endif /* MUSA_AITER_KV_PAGED_ATTENTION_H_ */
