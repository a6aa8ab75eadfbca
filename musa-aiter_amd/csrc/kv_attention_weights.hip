// The attention weight that cached tokens gather: kv_accumulate_attention_weights.
//
//   weights[b, h, j] += sum over the rows and heads of kv head h that see j of e^(s_j - lse)
//
// with the scores s_j of kv_cache_attention.hip and the logarithms it returned.  A token's sum is made by one
// workgroup, in the same order in every run: no atomics.
#include "kv_cache_attention.h"

namespace kvhip {
namespace catt {
namespace {

// ----- any shape and type: a thread per token, one row and head after the other --------------------
template <int DT>
__global__ __launch_bounds__(kBlockThreads) void weights_any_kernel(const CacheArgs a) {
  const AttnCall& c = a.r.c;
  const int32_t seq = blockIdx.y, head = blockIdx.z;
  const int64_t bs = a.r.bs, hd = a.r.hd;
  constexpr int64_t kElt = DT == kLinF32 ? 4 : 2;
  __shared__ float q[kVisitDims];
  const SeqRows rows = seq_rows(c, seq);
  if (rows.count == 0) return;
  const int32_t count = static_cast<int32_t>(rows.count);
  const View w = make_view(a, seq, count, 0, count - 1);
  for (int32_t base = blockIdx.x * kBlockThreads; base < w.length; base += gridDim.x * kBlockThreads) {
    const int32_t v = base + threadIdx.x;
    const int32_t token = position(w, v);
    int64_t k = -1;
    if (v < w.length && token < a.weight_tokens && (tile_bits(w, token) & 1u) != 0) {
      const int64_t blk = position_block(a, seq, token);
      if (blk >= 0) k = blk * (c.cache_block_stride[0] / kElt) + head * hd * bs + token % bs;
    }
    float sum = 0.0f;
    for (int32_t x = 0; x < count * a.r.group; ++x) {
      const int32_t i = x / a.r.group;
      const int64_t row = rows.first + i, hq = head * a.r.group + x % a.r.group;
      __syncthreads();
      for (int64_t d = threadIdx.x; d < hd; d += kBlockThreads)
        q[d] = load_q<DT>(c.query, row * c.query_row_stride + hq * c.query_head_stride + d);
      __syncthreads();
      const float lse = c.lse[row * c.heads + hq];
      if (lse == -__builtin_inff() || k < 0 || (row_bits(a, w, row_sight(a, w, 0, i), token) & 1u) == 0) continue;
      float dot = 0.0f;
      for (int64_t d = 0; d < hd; ++d) dot = __builtin_fmaf(q[d], load_q<DT>(c.cache[0], k + d * bs), dot);
      // The difference first: it is small where a weight is large, and its product then loses nothing.
      sum += __builtin_amdgcn_exp2f(__builtin_fmaf(dot, a.scale, -lse) * kLog2e);
    }
    if (k >= 0) {
      float* to = a.weights + seq * a.weight_row_stride + head * a.weight_head_stride + token;
      *to += sum;
    }
  }
}

template <int DT>
hipError_t launch(const CacheAttnCall& c, const CacheArgs& a, hipStream_t stream) {
  const int64_t room = c.max_blocks * c.block_size;
  int64_t longest = c.longest < room ? c.longest : room;
  if (longest > c.weight_tokens) longest = c.weight_tokens;
  int64_t groups = (longest + kBlockThreads - 1) / kBlockThreads;
  groups = groups < 1 ? 1 : groups < 4096 ? groups : 4096;
  weights_any_kernel<DT><<<dim3(groups, c.batch, c.kv_heads), kBlockThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace
}  // namespace catt

hipError_t launch_attention_weights(const CacheAttnCall& c, hipStream_t stream) {
  const catt::CacheArgs a = catt::cache_args(c, 0);
  switch (c.dtype) {
    case kLinF32: return catt::launch<kLinF32>(c, a, stream);
    case kLinF16: return catt::launch<kLinF16>(c, a, stream);
    default: return catt::launch<kLinBF16>(c, a, stream);
  }
}

}  // namespace kvhip
