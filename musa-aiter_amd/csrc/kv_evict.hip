// Eviction from a paged cache by gathered attention weight: kv_evict_paged_tokens.
//
// Two launches.  The first decides, one workgroup per line (a layer, row and kv head): a radix select finds the weight
// of the last token that stays, a pass in order marks the tokens (one bit each, in the workspace) and moves their
// weights.  The second moves the tokens' values.  A token's new position is never behind its old one, so a wave that
// goes through a line in order, with a step's loads ahead of its stores, can move it in place; lines and head
// dimensions are independent of each other.
#include "kv_cache_attention.h"

namespace kvhip {
namespace {

using attn::int_at;

struct EvictArgs {
  EvictCall c;
  int64_t words;  // of 64 positions, of a line
};

// Tokens that a line keeps, or -1 where it stays as it is.
__device__ __forceinline__ int64_t* line_keep(const EvictArgs& a, int64_t line) {
  return static_cast<int64_t*>(a.c.workspace) + line;
}
__device__ __forceinline__ uint64_t* line_bits(const EvictArgs& a, int64_t line) {
  return static_cast<uint64_t*>(a.c.workspace) + a.c.layers * a.c.batch * a.c.kv_heads + line * a.words;
}

__device__ __forceinline__ int64_t row_block(const EvictCall& c, int64_t row, int64_t token) {
  return int_at(c.tables, row * c.table_stride + token / c.block_size, c.wide_tables);
}

// Keys in the order of the weights: NaN below all others, the two zeros one.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u ^ ((u >> 31) != 0 ? 0xFFFFFFFFu : 0x80000000u);
}

constexpr int kDigit = 8;
constexpr int kBins = 1 << kDigit;
static_assert(kBins == kBlockThreads, "a thread per bin");

__global__ __launch_bounds__(kBlockThreads) void evict_select_kernel(const EvictArgs a) {
  const EvictCall& c = a.c;
  const int64_t line = blockIdx.x;
  const int64_t head = line % c.kv_heads, row = line / c.kv_heads % c.batch, layer = line / c.kv_heads / c.batch;
  const int lane = lane_id(), wave = wave_in_block();
  __shared__ int32_t bad;
  __shared__ uint32_t bins[kWavesPerBlock][kBins];
  __shared__ uint32_t above[kBins + 1];
  __shared__ uint32_t digit_found, need_left;
  __shared__ uint32_t more_of[kWavesPerBlock], same_of[kWavesPerBlock];

  const int64_t said = int_at(c.lens, row, c.wide_lens), asked = int_at(c.keep, row, c.wide_keep);
  const int64_t len = said < 0 ? 0 : said, room = c.max_blocks * c.block_size;
  if (threadIdx.x == 0) bad = asked < 0 || asked >= len || len > room ? 1 : 0;
  __syncthreads();
  if (bad == 0) {
    bool miss = false;
    for (int64_t p = threadIdx.x; p * c.block_size < len; p += kBlockThreads) {
      const int64_t blk = int_at(c.tables, row * c.table_stride + p, c.wide_tables);
      miss |= blk < 0 || blk >= c.num_blocks || (c.refs != nullptr && int_at(c.refs, blk, c.wide_refs) > 1);
    }
    if (miss) bad = 1;
  }
  __syncthreads();
  const bool stays = bad != 0;
  if (threadIdx.x == 0) {
    *line_keep(a, line) = stays ? -1 : asked;
    if (layer == 0 && head == 0) c.kept[row] = stays ? len : asked;
  }
  if (stays) return;

  const int64_t keep = asked;
  const int64_t first = c.sinks < keep ? c.sinks : keep;
  const int64_t recent = c.recent < keep - first ? c.recent : keep - first;
  const int64_t from = first, to = len - recent;  // where the heaviest are looked for
  float* weights = c.weights + layer * c.weight_layer_stride + row * c.weight_row_stride + head * c.weight_head_stride;
  auto weight_at = [&](int64_t p) { return p < c.weight_tokens ? weights[p] : 0.0f; };

  // The key of the lightest one that stays, digit by digit from the top, and how many of that key stay.
  uint32_t key = 0, need = static_cast<uint32_t>(keep - first - recent);
  const bool choose = need > 0;
  for (int shift = 32 - kDigit; choose && shift >= 0; shift -= kDigit) {
    for (int x = 0; x < kWavesPerBlock; ++x) bins[x][threadIdx.x] = 0;
    __syncthreads();
    for (int64_t p = from + threadIdx.x; p < to; p += kBlockThreads) {
      const uint32_t k = weight_key(weight_at(p));
      if (shift + kDigit == 32 || k >> (shift + kDigit) == key >> (shift + kDigit))
        atomicAdd(&bins[wave][k >> shift & (kBins - 1)], 1u);
    }
    __syncthreads();
    // above[t]: keys whose digit is t or more.
    uint32_t mine = 0;
    for (int x = 0; x < kWavesPerBlock; ++x) mine += bins[x][threadIdx.x];
    above[threadIdx.x] = mine;
    if (threadIdx.x == 0) above[kBins] = 0;
    __syncthreads();
    for (int o = 1; o < kBins; o <<= 1) {
      const uint32_t add = threadIdx.x + o < kBins ? above[threadIdx.x + o] : 0;
      __syncthreads();
      above[threadIdx.x] += add;
      __syncthreads();
    }
    const uint32_t next = above[threadIdx.x + 1];
    if (above[threadIdx.x] >= need && next < need) {
      digit_found = threadIdx.x;
      need_left = need - next;
    }
    __syncthreads();
    key |= digit_found << shift;
    need = need_left;
    __syncthreads();
  }

  // In order: the marks, and the weights to their new places.  `rank` tokens stay in front of a step, `same` of them
  // with the key itself.
  uint64_t* bits = line_bits(a, line);
  int64_t rank = 0;
  uint32_t same = 0;
  for (int64_t base = 0; base < len; base += kBlockThreads) {
    const int64_t p = base + threadIdx.x;
    const float weight = p < len ? weight_at(p) : 0.0f;
    const uint32_t k = weight_key(weight);
    const bool always = p < first || (p >= to && p < len), between = choose && p >= from && p < to;
    const uint64_t equal = ballot(between && k == key);
    if (lane == 0) same_of[wave] = __popcll(equal);
    __syncthreads();
    uint32_t in_front = same;
    for (int x = 0; x < kWavesPerBlock; ++x) {
      if (x < wave) in_front += same_of[x];
      same += same_of[x];
    }
    in_front += __popcll(equal & ((uint64_t{1} << lane) - 1));
    const bool stay = always || (between && (k > key || (k == key && in_front < need)));
    const uint64_t mark = ballot(stay);
    if (lane == 0) {
      more_of[wave] = __popcll(mark);
      if (base + wave * kWave < len) bits[(base >> 6) + wave] = mark;
    }
    __syncthreads();  // also: every weight of this step is read
    int64_t dst = rank + __popcll(mark & ((uint64_t{1} << lane) - 1));
    for (int x = 0; x < kWavesPerBlock; ++x) {
      if (x < wave) dst += more_of[x];
      rank += more_of[x];
    }
    if (stay && dst < c.weight_tokens) weights[dst] = weight;
  }
  for (int64_t p = keep + threadIdx.x; p < len && p < c.weight_tokens; p += kBlockThreads) weights[p] = 0.0f;
}

// ----- moving values, any element size and block size ----------------------------------------------
constexpr int kMoveDims = 8;  // head dimensions of a wave

template <int ELT>
__global__ __launch_bounds__(kBlockThreads) void evict_move_any_kernel(const EvictArgs a) {
  const EvictCall& c = a.c;
  using T = typename VecType<ELT>::T;
  const int64_t line = blockIdx.x;
  const int kv = blockIdx.z;
  const int64_t keep = uniform64(*line_keep(a, line));
  const int64_t d0 = (static_cast<int64_t>(blockIdx.y) * kWavesPerBlock + wave_in_block()) * kMoveDims;
  if (keep < 0 || d0 >= c.head_dim) return;
  const int64_t head = line % c.kv_heads, row = line / c.kv_heads % c.batch, layer = line / c.kv_heads / c.batch;
  const int64_t bs = c.block_size;
  uint8_t* base = static_cast<uint8_t*>(c.cache[kv]) + layer * c.cache_layer_stride[kv] +
                  (head * c.head_dim + d0) * bs * ELT;
  const int dims = static_cast<int>(c.head_dim - d0 < kMoveDims ? c.head_dim - d0 : kMoveDims);
  const uint64_t* bits = line_bits(a, line);
  auto place = [&](int64_t token) {
    const int64_t blk = row_block(c, row, token);
    return base + blk * c.cache_block_stride[kv] + token % bs * ELT;
  };
  int64_t rank = 0;
  for (int64_t word = 0; rank < keep; ++word) {
    const uint64_t mark = static_cast<uint64_t>(uniform64(static_cast<int64_t>(bits[word])));
    const int64_t src = word * kWave + lane_id();
    const int64_t dst = rank + __popcll(mark & ((uint64_t{1} << lane_id()) - 1));
    rank += __popcll(mark);
    if ((mark >> lane_id() & 1) == 0 || src == dst) continue;
    const uint8_t* in = place(src);
    uint8_t* out = place(dst);
    T value[kMoveDims];
#pragma unroll
    for (int d = 0; d < kMoveDims; ++d)
      if (d < dims) value[d] = *reinterpret_cast<const KVHIP_GLOBAL T*>(reinterpret_cast<uint64_t>(in + d * bs * ELT));
#pragma unroll
    for (int d = 0; d < kMoveDims; ++d)
      if (d < dims) *reinterpret_cast<KVHIP_GLOBAL T*>(reinterpret_cast<uint64_t>(out + d * bs * ELT)) = value[d];
  }
}

EvictArgs evict_args(const EvictCall& c) {
  EvictArgs a{};
  a.c = c;
  a.words = (c.max_blocks * c.block_size + kWave - 1) / kWave;
  return a;
}

}  // namespace

int64_t evict_workspace(const EvictCall& c) {
  return c.layers * c.batch * c.kv_heads * (evict_args(c).words + 1) * 8;
}

hipError_t launch_evict(const EvictCall& c, hipStream_t stream) {
  const EvictArgs a = evict_args(c);
  const int64_t lines = c.layers * c.batch * c.kv_heads;
  evict_select_kernel<<<dim3(lines), kBlockThreads, 0, stream>>>(a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const int64_t slices = (c.head_dim + kMoveDims * kWavesPerBlock - 1) / (kMoveDims * kWavesPerBlock);
  const dim3 grid(lines, slices, 2);
  if (c.element_bytes == 1) evict_move_any_kernel<1><<<grid, kBlockThreads, 0, stream>>>(a);
  else if (c.element_bytes == 2) evict_move_any_kernel<2><<<grid, kBlockThreads, 0, stream>>>(a);
  else evict_move_any_kernel<4><<<grid, kBlockThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace kvhip
