// C-ABI of the operators on paged caches that are not copies (include/musa_aiter_kv_serving.h): argument
// checks, then the launchers of kv_block_store.hip, kv_attention.hip and kv_pages.hip.
#include <climits>

#include "kv_host_calls.h"
#include "kv_host_wait.h"
#include "kv_serving.h"

namespace {

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr int64_t kMaxExtent = int64_t{1} << 31;
bool extent(int64_t v, int64_t least) { return v >= least && v < kMaxExtent; }

constexpr int64_t kCheckPerGroup = 1024;  // slots per workgroup of the check kernel

int block_store(const musa_aiter_hip_block_store_call& c, hipStream_t stream) {
  if (!extent(c.num_layers, 0) || !extent(c.num_tokens, 0) || !extent(c.num_blocks, 1) || !extent(c.num_heads, 1) ||
      !extent(c.head_dim, 1) || !extent(c.block_size, 1) || c.num_layers > 65535 || c.num_heads > 65535 ||
      (c.codec != kvhip::kE4M3 && c.codec != kvhip::kE5M2) || c.lin_dtype < 0 || c.lin_dtype > 2)
    return hipErrorInvalidValue;
  if (c.num_layers == 0 || c.num_tokens == 0) return hipSuccess;
  if (c.slots == nullptr || (c.report != nullptr && (c.guard == nullptr || c.report_words < 1 || c.stamp <= 0)))
    return hipErrorInvalidValue;
  kvhip::BlockStoreParams p{};
  for (int kv = 0; kv < 2; ++kv) {
    if (c.linear[kv] == nullptr || c.cache[kv] == nullptr || c.scale[kv] == nullptr) return hipErrorInvalidValue;
    p.lin[kv] = c.linear[kv];
    p.cache[kv] = static_cast<uint8_t*>(c.cache[kv]);
    p.scale[kv] = c.scale[kv];
    p.block_stride[kv] = c.cache_block_stride[kv];
    p.layer_stride[kv] = c.cache_layer_stride[kv];
  }
  p.slots = c.slots;
  p.codec = c.codec;
  p.lin_dtype = c.lin_dtype;
  p.num_layers = c.num_layers;
  p.num_tokens = c.num_tokens;
  p.num_blocks = c.num_blocks;
  p.num_heads = c.num_heads;
  p.head_dim = c.head_dim;
  p.block_size = c.block_size;
  p.lin_token_stride = c.lin_token_stride;
  p.lin_layer_stride = c.lin_layer_stride;
  p.check.stamp = c.stamp;
  bool refused = false;
  if (c.num_tokens <= kvhip::kStoreScanTokens && c.block_size <= kvhip::kStoreScanColumns) {
    // Every workgroup reads all slots, finds its block's columns among them and refuses the call by itself.
    p.check.report = c.report;
    hipError_t err = kvhip::launch_block_store(p, stream);
    if (err != hipSuccess || c.report == nullptr) return err;
    err = kvhip::await_verdict(c.report, 1, c.stamp, stream, &refused);
    return err != hipSuccess ? err : refused ? MUSA_AITER_HIP_REFUSED : 0;
  }
  const int64_t rows = c.num_blocks * c.block_size;
  if (c.claims == nullptr || c.claims->tags == nullptr || c.claims->capacity < rows) return hipErrorInvalidValue;
  p.owner = c.claims->tags;
  if (c.report == nullptr || c.claims->epoch == 0) {
    // No verdict: a call that is captured, whose replays repeat the epoch, so the tags are cleared first.
    if (c.report != nullptr) return hipErrorInvalidValue;
    p.epoch = 1;
    hipError_t err = kvhip::launch_block_tag_reset(c.slots, c.num_tokens, c.num_blocks, c.block_size,
                                                   c.claims->tags, stream);
    kvhip::ClaimSource src;
    src.idx = c.slots;
    if (err == hipSuccess) err = kvhip::launch_claim(src, c.num_tokens, rows, c.claims->tags, 1, stream);
    return err != hipSuccess ? err : kvhip::launch_block_store(p, stream);
  }
  kvhip::CheckSource src{};
  src.idx = c.slots;
  src.n = c.num_tokens;
  src.rows = rows;
  src.low = INT64_MIN;
  src.owner = c.claims->tags;
  src.epoch = p.epoch = c.claims->epoch;
  int64_t groups = (c.num_tokens + kCheckPerGroup - 1) / kCheckPerGroup;
  if (groups > c.report_words) groups = c.report_words;
  const kvhip::CallCheck check{c.report, c.guard, c.stamp, 0};
  hipError_t err = kvhip::launch_check(src, check, groups, stream);
  if (err != hipSuccess) return err;
  p.check.guard = c.guard;
  const hipError_t stored = kvhip::launch_block_store(p, stream);
  err = kvhip::await_verdict(c.report, groups, c.stamp, stream, &refused);
  if (err != hipSuccess || refused) return err != hipSuccess ? err : MUSA_AITER_HIP_REFUSED;
  return stored;
}

bool attention_sizes_ok(const musa_aiter_hip_attention_call& c) {
  return extent(c.rows, 0) && extent(c.batch, 0) && extent(c.heads, 1) && extent(c.kv_heads, 1) &&
         extent(c.head_dim, 1) && extent(c.block_size, 1) && extent(c.num_blocks, 1) && extent(c.max_blocks, 0) &&
         c.heads % c.kv_heads == 0 && c.heads <= 65535 && c.head_dim <= 512 && c.window >= 0 &&
         c.rows * c.heads < kMaxExtent && c.max_blocks * c.block_size <= kMaxExtent / 4;
}

int attention(const musa_aiter_hip_attention_call& c, hipStream_t stream) {
  if (!attention_sizes_ok(c) || c.dtype < 0 || c.dtype > 2 || (c.codec != kvhip::kE4M3 && c.codec != kvhip::kE5M2) ||
      c.splits < 0 || c.splits > 64)
    return hipErrorInvalidValue;
  if (c.rows == 0) return hipSuccess;
  if (c.query == nullptr || c.out == nullptr || (c.batch > 0 && c.lens == nullptr) ||
      (c.batch > 0 && c.max_blocks > 0 && c.tables == nullptr))
    return hipErrorInvalidValue;
  if (c.starts == nullptr && c.rows != c.batch) return hipErrorInvalidValue;
  for (int kv = 0; kv < 2; ++kv)
    if (c.cache[kv] == nullptr || c.scale[kv] == nullptr) return hipErrorInvalidValue;
  if (c.splits == 0 && !kvhip::attention_flows(c)) return hipErrorInvalidValue;
  if (c.workspace_bytes < kvhip::attention_workspace(c) || (c.splits != 1 && c.workspace == nullptr))
    return hipErrorInvalidValue;
  return kvhip::launch_attention(c, stream);
}

}  // namespace

extern "C" {

int musa_aiter_hip_block_store(const musa_aiter_hip_block_store_call* call, void* stream) {
  return call == nullptr ? hipErrorInvalidValue : block_store(*call, as_stream(stream));
}

int musa_aiter_hip_attention(const musa_aiter_hip_attention_call* call, void* stream) {
  return call == nullptr ? hipErrorInvalidValue : attention(*call, as_stream(stream));
}

int64_t musa_aiter_hip_attention_splits(const musa_aiter_hip_attention_call* call, int64_t longest) {
  return call == nullptr || !attention_sizes_ok(*call) ? 1 : kvhip::attention_splits(*call, longest);
}

int64_t musa_aiter_hip_attention_workspace(const musa_aiter_hip_attention_call* call) {
  return call == nullptr || !attention_sizes_ok(*call) ? 0 : kvhip::attention_workspace(*call);
}

int musa_aiter_hip_pages_free(const musa_aiter_hip_pages_call* call, void* stream) {
  return call == nullptr ? hipErrorInvalidValue : kvhip::launch_pages(*call, kvhip::kPagesFree, as_stream(stream));
}

int musa_aiter_hip_pages_fork(const musa_aiter_hip_pages_call* call, void* stream) {
  return call == nullptr ? hipErrorInvalidValue : kvhip::launch_pages(*call, kvhip::kPagesFork, as_stream(stream));
}

int musa_aiter_hip_pages_extend(const musa_aiter_hip_pages_call* call, void* stream) {
  return call == nullptr ? hipErrorInvalidValue : kvhip::launch_pages(*call, kvhip::kPagesExtend, as_stream(stream));
}

int musa_aiter_hip_pages_compact(const musa_aiter_hip_pages_call* call, void* stream) {
  return call == nullptr ? hipErrorInvalidValue : kvhip::launch_pages(*call, kvhip::kPagesCompact, as_stream(stream));
}

int64_t musa_aiter_hip_pages_workspace(const musa_aiter_hip_pages_call* call, int64_t kind) {
  if (call == nullptr || call->batch < 0 || call->max_blocks < 0 || call->num_blocks < 0 || kind < 0 || kind > 2)
    return 0;
  return kvhip::pages_workspace(*call, static_cast<kvhip::PagesKind>(kind));
}

}  // extern "C"
