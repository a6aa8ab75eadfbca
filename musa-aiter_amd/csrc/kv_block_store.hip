// FP8 store into paged caches with one scale per (block, head): kv_linear_to_paged_fp8_block.
//
// Per layer, block b, kv head h and plane, with N the finite new values of the block and F the format's
// largest value (448 / 57344):
//   anew = column 0 is written, or the old scale is not positive and finite
//   s    = max(max|N| / F, 2^-60, anew ? 0 : s_old)
//   written column: encode(x / s);  other columns: 0 if anew, as they are if s == s_old, else
//   encode(decode(code) * s_old / s)
// all in fp32 with one rounding per operation, so the result does not depend on how the work is cut.
//
// The tokens of a block may stand anywhere in the call.  One wave has one (block, plane, head, layer): the
// block's leader, the token that owns the lowest written column, names the block, and the columns' tokens come
// from the claim tags of the call (or, for few tokens, from the slots themselves, read by every workgroup).
#include "kv_serving.h"

namespace kvhip {
namespace {

template <int CODEC>
constexpr float kCodecMax = CODEC == kE4M3 ? 448.0f : 57344.0f;

struct StoreArgs {
  BlockStoreParams p;
};

// Token that writes column `col` of `block`, or -1.
__device__ __forceinline__ int64_t column_token(const BlockStoreParams& p, const int64_t* scan, int64_t block,
                                                int64_t col) {
  const int64_t slot = block * p.block_size + col;
  if (p.owner != nullptr) {
    const uint64_t tag = p.owner[slot];
    return static_cast<uint32_t>(tag >> 32) == p.epoch ? static_cast<int64_t>(tag & 0xFFFFFFFFu) - 1 : -1;
  }
  int64_t found = -1;
  for (int64_t t = 0; t < p.num_tokens; ++t)
    if (scan[t] == slot) found = t;
  return found;
}

template <int LDT>
__device__ __forceinline__ float load_lin(const void* base, int64_t i) {
  if constexpr (LDT == kLinF32) return static_cast<const float*>(base)[i];
  else return lin_to_f32<LDT>(static_cast<const uint16_t*>(base)[i]);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// One wave per (token, plane, head, layer); waves whose token leads no block end at once.
template <int CODEC, int LDT>
__global__ __launch_bounds__(kBlockThreads) void block_store_kernel(const StoreArgs a) {
  const BlockStoreParams& p = a.p;
  __shared__ int64_t scan[kStoreScanTokens];
  __shared__ int refused;
  if (refused_ahead(p.check)) return;
  const int64_t slots_all = p.num_blocks * p.block_size;
  if (p.owner == nullptr) {
    if (threadIdx.x == 0) refused = 0;
    __syncthreads();
    for (int64_t t = threadIdx.x; t < p.num_tokens; t += kBlockThreads) {
      const int64_t s = p.slots[t];
      scan[t] = s;
      if (s >= slots_all) refused = 1;
    }
    __syncthreads();
    if (p.check.report != nullptr) {
      if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0)
        __hip_atomic_store(p.check.report, 2 * p.check.stamp + refused, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
      if (refused) return;
    }
  }
  const int64_t t = blockIdx.x;
  const int64_t unit = static_cast<int64_t>(blockIdx.y) * kWavesPerBlock + wave_in_block();
  if (unit >= 2 * p.num_heads) return;
  const int64_t layer = blockIdx.z;
  const int kv = static_cast<int>(unit & 1);
  const int64_t head = unit >> 1;
  const int64_t slot = p.slots[t];
  if (slot < 0 || slot >= slots_all) return;
  const int64_t block = slot / p.block_size, bs = p.block_size;
  // Leader: this token owns its column, and no lower column is written.
  bool leads = true;
  for (int64_t c0 = 0; c0 <= slot - block * bs && leads; c0 += kWave) {
    const int64_t col = c0 + lane_id();
    const int64_t owner = col <= slot - block * bs ? column_token(p, scan, block, col) : -1;
    leads = ballot(col < slot - block * bs ? owner >= 0 : col == slot - block * bs && owner != t) == 0;
  }
  if (!leads) return;

  const void* lin = p.lin[kv];
  const int64_t lin0 = layer * p.lin_layer_stride + head * p.head_dim;
  uint8_t* codes = p.cache[kv] + layer * p.layer_stride[kv] + block * p.block_stride[kv] + head * p.head_dim * bs;
  float* scale = p.scale[kv] + (layer * p.num_blocks + block) * p.num_heads + head;
  float most = 0.0f;
  for (int64_t col = 0; col < bs; ++col) {
    const int64_t tok = column_token(p, scan, block, col);
    if (tok < 0) continue;
    for (int64_t d = lane_id(); d < p.head_dim; d += kWave) {
      const float x = fabsf(load_lin<LDT>(lin, lin0 + tok * p.lin_token_stride + d));
      most = fmaxf(most, x < __builtin_inff() ? x : 0.0f);
    }
  }
  most = wave_max(most);
  const float before = *scale;
  const bool anew = slot == block * bs || scale_refused(before);
  float now = fmaxf(div_rn(most, kCodecMax<CODEC>), kScaleFloor);
  if (!anew) now = fmaxf(now, before);
  for (int64_t col = 0; col < bs; ++col) {
    const int64_t tok = column_token(p, scan, block, col);
    if (tok < 0 && !anew && now == before) continue;
    for (int64_t d = lane_id(); d < p.head_dim; d += kWave) {
      uint8_t* at = codes + d * bs + col;
      uint32_t code = 0;
      if (tok >= 0) code = fp8_encode<CODEC>(div_rn(load_lin<LDT>(lin, lin0 + tok * p.lin_token_stride + d), now));
      else if (!anew) code = fp8_encode<CODEC>(div_rn(fp8_decode<CODEC>(*at) * before, now));
      *at = static_cast<uint8_t>(code);
    }
  }
  if (lane_id() == 0) *scale = now;
}

__global__ __launch_bounds__(kBlockThreads) void block_tag_reset_kernel(const int64_t* slots, int64_t n,
                                                                        int64_t num_blocks, int64_t bs,
                                                                        uint64_t* owner) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlockThreads + threadIdx.x;
  const int64_t t = i / bs;
  if (t >= n) return;
  const int64_t s = slots[t];
  if (s < 0 || s >= num_blocks * bs) return;
  owner[s / bs * bs + (i - t * bs)] = 0;
}

template <int CODEC, int LDT>
hipError_t launch_typed(const BlockStoreParams& p, hipStream_t stream) {
  const StoreArgs a{p};
  const dim3 grid(static_cast<uint32_t>(p.num_tokens),
                  static_cast<uint32_t>((2 * p.num_heads + kWavesPerBlock - 1) / kWavesPerBlock),
                  static_cast<uint32_t>(p.num_layers));
  hipLaunchKernelGGL(HIP_KERNEL_NAME(block_store_kernel<CODEC, LDT>), grid, dim3(kBlockThreads), 0, stream, a);
  return hipGetLastError();
}

template <int CODEC>
hipError_t launch_codec(const BlockStoreParams& p, hipStream_t stream) {
  switch (p.lin_dtype) {
    case kLinF32: return launch_typed<CODEC, kLinF32>(p, stream);
    case kLinF16: return launch_typed<CODEC, kLinF16>(p, stream);
    case kLinBF16: return launch_typed<CODEC, kLinBF16>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_block_store(const BlockStoreParams& p, hipStream_t stream) {
  if (p.owner == nullptr && p.num_tokens > kStoreScanTokens) return hipErrorInvalidValue;
  return p.codec == kE4M3 ? launch_codec<kE4M3>(p, stream)
         : p.codec == kE5M2 ? launch_codec<kE5M2>(p, stream) : hipErrorInvalidValue;
}

hipError_t launch_block_tag_reset(const int64_t* slots, int64_t n, int64_t num_blocks, int64_t block_size,
                                  uint64_t* owner, hipStream_t stream) {
  const int64_t groups = (n * block_size + kBlockThreads - 1) / kBlockThreads;
  if (groups < 1 || groups >= int64_t{1} << 31) return hipErrorInvalidValue;
  hipLaunchKernelGGL(block_tag_reset_kernel, dim3(static_cast<uint32_t>(groups)), dim3(kBlockThreads), 0, stream, slots,
                     n, num_blocks, block_size, owner);
  return hipGetLastError();
}

}  // namespace kvhip
