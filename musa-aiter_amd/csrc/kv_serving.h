// Host-side launcher interfaces of the operators on paged caches that are not copies (the block-scaled FP8
// store, the attention over it, the page bookkeeping).  Nothing here is exported from the shared library.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_launch.h"
#include "musa_aiter_kv_serving.h"

namespace kvhip {

// The smallest scale a store gives a block: below it a quotient would leave the range of the codec's fast
// division (see quot_fast).  Values under 448 * 2^-60 lose bits to it.
constexpr float kScaleFloor = 0x1p-60f;

struct BlockStoreParams {
  const void* lin[2];
  uint8_t* cache[2];
  float* scale[2];
  const int64_t* slots;
  const uint64_t* owner;  // claim tags of `epoch` over the caches' slots (null: the kernel scans the slots)
  uint32_t epoch;
  int codec;
  int lin_dtype;
  int64_t num_layers, num_tokens, num_blocks, num_heads, head_dim, block_size;
  int64_t lin_token_stride, lin_layer_stride;        // elements
  int64_t block_stride[2], layer_stride[2];          // bytes
  CallCheck check;
};

// Tokens of a store that finds its blocks' columns by reading all slots in the kernel (one launch, a thread per
// slot), and columns of a block that it has place for.
constexpr int64_t kStoreScanTokens = 256;
constexpr int64_t kStoreScanColumns = 1024;

hipError_t launch_block_store(const BlockStoreParams& p, hipStream_t stream);
// Zeroes the tags of every column of the blocks that the tokens write (calls captured into graphs).
hipError_t launch_block_tag_reset(const int64_t* slots, int64_t n, int64_t num_blocks, int64_t block_size,
                                  uint64_t* owner, hipStream_t stream);

hipError_t launch_attention(const musa_aiter_hip_attention_call& c, hipStream_t stream);
// Whether the call can be cut evenly (splits 0).
bool attention_flows(const musa_aiter_hip_attention_call& c);
int64_t attention_splits(const musa_aiter_hip_attention_call& c, int64_t longest);
int64_t attention_workspace(const musa_aiter_hip_attention_call& c);

enum PagesKind : int { kPagesFork = 0, kPagesExtend = 1, kPagesCompact = 2, kPagesFree = 3 };
hipError_t launch_pages(const musa_aiter_hip_pages_call& c, PagesKind kind, hipStream_t stream);
int64_t pages_workspace(const musa_aiter_hip_pages_call& c, PagesKind kind);

}  // namespace kvhip
