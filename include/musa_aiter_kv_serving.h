/*
 * C-ABI of libmusa_aiter_kv_hip.so, second part: operators on paged caches that are not copies -- the FP8
 * store with one scale per block and head, the attention over such a cache, and the bookkeeping of pages.
 * None of them has a reference counterpart.
 *
 * As in musa_aiter_kv_hip.h every entry launches asynchronously on `stream` and returns the HIP status (or
 * MUSA_AITER_HIP_REFUSED where it says so); nothing is launched for arguments that are refused.  Device
 * tables, lengths, slots and reference counts are read on the device only, and every id read from them is
 * checked there before it is used as an address.
 */
#ifndef MUSA_AITER_KV_SERVING_H_
#define MUSA_AITER_KV_SERVING_H_

#include <stdint.h>

#include "musa_aiter_kv_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- FP8 store with one scale per (block, head) -------------------------------------------------
 * Caches [layers, blocks, heads, head_dim, block_size] of codes, scales float32 [layers, blocks, heads]
 * (contiguous).  Per layer, block, head and plane (K, V): scale = max(max|finite new| / F, 2^-60, old scale),
 * F = 448 (E4M3) or 57344 (E5M2); other columns are encoded anew where the scale grew.  A call that writes
 * column 0, or that meets a scale that is not positive and finite, starts the block anew: the old scale does
 * not count and columns that are not written become 0.  A slot named twice keeps the last token; slots < 0
 * are skipped.
 * lin_dtype: 0 f32, 1 f16, 2 bf16; strides in elements (rows of [heads, head_dim] packed); block strides in
 * bytes.  claims: tags for num_blocks * block_size slots, as musa_aiter_hip_claims describes.
 * report / guard / stamp as in musa_aiter_hip_paged_tiles_checked: slots past the cache are refused
 * (MUSA_AITER_HIP_REFUSED, nothing stored); with report NULL they are skipped. */
typedef struct musa_aiter_hip_block_store_call {
  const void* linear[2];
  void* cache[2];
  float* scale[2];
  const int64_t* slots;
  const musa_aiter_hip_claims* claims;
  int64_t* report;
  int64_t* guard;
  int64_t stamp;
  int64_t report_words;
  int64_t num_layers, num_tokens, num_blocks, num_heads, head_dim, block_size;
  int64_t lin_token_stride, lin_layer_stride;
  int64_t cache_block_stride[2], cache_layer_stride[2];
  int32_t codec;
  int32_t lin_dtype;
} musa_aiter_hip_block_store_call;
int musa_aiter_hip_block_store(const musa_aiter_hip_block_store_call* call, void* stream);

/* ---- Attention over an FP8 cache with one scale per (block, head) --------------------------------
 * query / out [rows, heads, head_dim] (dtype 0 f32, 1 f16, 2 bf16; out packed), lse float32 [rows, heads] or
 * NULL.  tables [batch, max_blocks], lens [batch], starts [batch + 1] or NULL (rows == batch, one row each);
 * wide flags: 1 int64, 0 int32.  Row i of the n of a sequence of `len` cached tokens sees positions
 * (len - n + i - window, len - n + i] (window 0: all up to it); positions whose table entry is missing or
 * outside the cache are not seen; a row that sees nothing gives 0 and lse -inf.  Rows of no sequence are
 * zeroed in out with fill_rows, else left as they are there; their lse is -inf.  Scales of blocks that rows
 * see are 0 or lie in [2^-60, 2^60]; query values are at most 2^100 in size, and E4M3 value scales at most 4
 * where a row's scores pass 2^24.
 * splits (1 to 64) parts of each sequence run side by side; 0 cuts the sequences of a decode step (starts NULL,
 * 16-bit queries, head_dim <= 256, blocks of multiples of 16 tokens at 16-byte addresses) into even shares of
 * the chip.  Unless splits is 1, `workspace` holds musa_aiter_hip_attention_workspace bytes. */
typedef struct musa_aiter_hip_attention_call {
  const void* query;
  void* out;
  float* lse;
  const void* cache[2];
  const float* scale[2];
  const void* tables;
  const void* lens;
  const void* starts;
  void* workspace;
  int64_t workspace_bytes;
  int64_t rows, batch, heads, kv_heads, head_dim, block_size, num_blocks, max_blocks;
  int64_t query_row_stride, query_head_stride;             /* elements */
  int64_t cache_block_stride[2];                            /* bytes */
  int64_t scale_block_stride[2], scale_head_stride[2];      /* elements */
  int64_t table_stride;                                     /* elements between rows of tables */
  int64_t window;
  int64_t splits;
  double softmax_scale;
  int32_t dtype;
  int32_t codec;
  int32_t wide_tables, wide_lens, wide_starts;
  int32_t fill_rows;
} musa_aiter_hip_attention_call;
int musa_aiter_hip_attention(const musa_aiter_hip_attention_call* call, void* stream);
/* Parts that each sequence of at most `longest` tokens is best cut into, and the workspace they need. */
int64_t musa_aiter_hip_attention_splits(const musa_aiter_hip_attention_call* call, int64_t longest);
int64_t musa_aiter_hip_attention_workspace(const musa_aiter_hip_attention_call* call);

/* ---- Bookkeeping of pages ------------------------------------------------------------------------
 * tables [batch, max_blocks] (table_stride elements between rows), lens [batch], refs [num_blocks]: int64 with
 * `wide`, else int32, contiguous but for the rows.  A sequence owns the first ceil(len / block_size) entries
 * of its row; refs counts a page's owners (0: free).  cache [layers, blocks, ...] of block_bytes per block with
 * strides in bytes; scale (nullable pair) float32 [layers, blocks, scale_values]. */
typedef struct musa_aiter_hip_pages_call {
  void* tables;
  void* lens;
  void* refs;
  const void* rows;     /* per row: parents (fork), tokens kept (free), new tokens (extend) */
  int64_t* slots;       /* extend: [batch, max_new] */
  int64_t* result;      /* extend: free pages left, -(pages missing), or -2^62 (a row outgrows its table
                           or the type of lens);
                           compact: pages in use */
  void* workspace;
  int64_t workspace_bytes;
  void* cache[2];
  float* scale[2];
  int64_t batch, max_blocks, table_stride, num_blocks, block_size, max_new;
  int64_t layers, block_bytes, block_stride[2], layer_stride[2];
  int64_t scale_values;
  int32_t wide;
  int32_t wide_rows;    /* rows holds int64 */
} musa_aiter_hip_pages_call;
int musa_aiter_hip_pages_free(const musa_aiter_hip_pages_call* call, void* stream);
int musa_aiter_hip_pages_fork(const musa_aiter_hip_pages_call* call, void* stream);
int musa_aiter_hip_pages_extend(const musa_aiter_hip_pages_call* call, void* stream);
int musa_aiter_hip_pages_compact(const musa_aiter_hip_pages_call* call, void* stream);
/* Workspace bytes: fork 0, extend 1, compact 2. */
int64_t musa_aiter_hip_pages_workspace(const musa_aiter_hip_pages_call* call, int64_t kind);

#ifdef __cplusplus
}
#endif

#endif /* MUSA_AITER_KV_SERVING_H_ */
