// C-ABI of the operators on paged caches of plain values (include/musa_aiter_kv_paged_attention.h): argument checks,
// then the launchers of kv_cache_attention.hip, kv_attention_weights.hip and kv_evict.hip.
#include "kv_cache_attention.h"

namespace {

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr int64_t kMaxExtent = int64_t{1} << 31;
constexpr int64_t kMaxRoom = int64_t{1} << 29;
bool extent(int64_t v, int64_t least) { return v >= least && v < kMaxExtent; }

bool table_ok(int64_t batch, int64_t max_blocks, int64_t block_size, int64_t num_blocks) {
  return extent(batch, 0) && extent(max_blocks, 0) && extent(block_size, 1) && extent(num_blocks, 1) &&
         max_blocks * block_size <= kMaxRoom;
}

bool sizes_ok(const kvhip::CacheAttnCall& c) {
  return table_ok(c.batch, c.max_blocks, c.block_size, c.num_blocks) && extent(c.rows, 0) && extent(c.heads, 1) &&
         extent(c.kv_heads, 1) && extent(c.head_dim, 1) && c.heads % c.kv_heads == 0 && c.heads <= 65535 &&
         c.head_dim <= 512 && c.rows <= kMaxRoom && c.rows * c.heads < kMaxExtent && c.window >= 0 && c.sinks >= 0 &&
         c.longest >= 0 && c.mask_words >= 0 && c.mask_words < kMaxExtent;
}

bool call_ok(const kvhip::CacheAttnCall& c) {
  if (!sizes_ok(c) || c.dtype < 0 || c.dtype > 2) return false;
  if (c.rows == 0) return true;
  if (c.query == nullptr || c.cache[0] == nullptr || (c.batch > 0 && c.lens == nullptr) ||
      (c.batch > 0 && c.max_blocks > 0 && c.tables == nullptr))
    return false;
  if (c.masks != nullptr && (c.mask_words < 1 || c.window != 0 || c.sinks != 0)) return false;
  return c.starts != nullptr || c.rows == c.batch;
}

int attention(const kvhip::CacheAttnCall& c, hipStream_t stream) {
  if (!call_ok(c)) return hipErrorInvalidValue;
  if (c.rows == 0) return hipSuccess;
  if (c.out == nullptr || c.cache[1] == nullptr) return hipErrorInvalidValue;
  const int64_t bytes = kvhip::cache_attention_workspace(c);
  if (bytes > 0 && (c.workspace == nullptr || c.workspace_bytes < bytes)) return hipErrorInvalidValue;
  return kvhip::launch_cache_attention(c, stream);
}

int attention_weights(const kvhip::CacheAttnCall& c, hipStream_t stream) {
  if (!call_ok(c) || c.masks != nullptr || c.weight_tokens < 0 || c.batch > 65535 || c.kv_heads > 65535)
    return hipErrorInvalidValue;
  if (c.rows == 0 || c.batch == 0 || c.weight_tokens == 0) return hipSuccess;
  if (c.lse == nullptr || c.weights == nullptr) return hipErrorInvalidValue;
  return kvhip::launch_attention_weights(c, stream);
}

bool evict_sizes_ok(const kvhip::EvictCall& c) {
  return table_ok(c.batch, c.max_blocks, c.block_size, c.num_blocks) && extent(c.layers, 1) && extent(c.kv_heads, 1) &&
         extent(c.head_dim, 1) && c.layers * c.batch < kMaxExtent && c.layers * c.batch * c.kv_heads < kMaxExtent &&
         c.head_dim <= 65535 && (c.element_bytes == 1 || c.element_bytes == 2 || c.element_bytes == 4);
}

int evict(const kvhip::EvictCall& c, hipStream_t stream) {
  if (!evict_sizes_ok(c) || c.weight_tokens < 0 || c.sinks < 0 || c.recent < 0) return hipErrorInvalidValue;
  if (c.batch == 0) return hipSuccess;
  if (c.cache[0] == nullptr || c.cache[1] == nullptr || c.lens == nullptr || c.keep == nullptr || c.kept == nullptr ||
      (c.max_blocks > 0 && c.tables == nullptr) || (c.weight_tokens > 0 && c.weights == nullptr) ||
      c.workspace == nullptr || c.workspace_bytes < kvhip::evict_workspace(c))
    return hipErrorInvalidValue;
  return kvhip::launch_evict(c, stream);
}

}  // namespace

extern "C" {

int musa_aiter_hip_paged_attention(const musa_aiter_hip_paged_attention_call* call, void* stream) {
  return call == nullptr ? hipErrorInvalidValue : attention(*call, as_stream(stream));
}

int64_t musa_aiter_hip_paged_attention_workspace(const musa_aiter_hip_paged_attention_call* call) {
  return call == nullptr || !sizes_ok(*call) || call->rows == 0 ? 0 : kvhip::cache_attention_workspace(*call);
}

int musa_aiter_hip_attention_weights(const musa_aiter_hip_paged_attention_call* call, void* stream) {
  return call == nullptr ? hipErrorInvalidValue : attention_weights(*call, as_stream(stream));
}

int musa_aiter_hip_evict(const musa_aiter_hip_evict_call* call, void* stream) {
  return call == nullptr ? hipErrorInvalidValue : evict(*call, as_stream(stream));
}

int64_t musa_aiter_hip_evict_workspace(const musa_aiter_hip_evict_call* call) {
  return call == nullptr || !evict_sizes_ok(*call) ? 0 : kvhip::evict_workspace(*call);
}

}  // extern "C"
