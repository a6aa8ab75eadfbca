// Eviction from a paged cache by gathered attention weight: kv_evict_paged_tokens.
//
// Two launches.  The first decides, one workgroup per line (a layer, row and kv head): a radix select finds the weight
// of the lightest token that stays, then the tokens are marked (one bit each, in the workspace) and their weights moved.
// The second moves the tokens' values.  A token's new position is never behind its old one, so a wave that goes through a
// line in order, with a step's loads ahead of its stores, can move it in place; lines and head dimensions are independent
// of each other.
//
// 8 sequences of 1520 to 6000 tokens to 1024 in 8 layers (8 heads of 128 dims, bf16): decisions 33 us, moves 279 (4.2 TB/s
// of the pages read and written).  One sequence of 40001 tokens to 8000 in two layers: 72 (16 workgroups) and 118.
#include "kv_cache_attention.h"

namespace kvhip {
namespace {

using attn::int_at;

struct EvictArgs {
  EvictCall c;
  int64_t words;  // of 64 positions, of a line
  int64_t lines;
};

// Tokens that a line keeps, or -1 where it stays as it is.
__device__ __forceinline__ int64_t* line_keep(const EvictArgs& a, int64_t line) {
  return static_cast<int64_t*>(a.c.workspace) + line;
}
__device__ __forceinline__ uint64_t* line_bits(const EvictArgs& a, int64_t line) {
  return static_cast<uint64_t*>(a.c.workspace) + a.lines + line * a.words;
}
// The weights of the tokens that stay, until all of the old ones are read.
__device__ __forceinline__ float* line_weights(const EvictArgs& a, int64_t line) {
  return reinterpret_cast<float*>(line_bits(a, a.lines)) + line * a.words * kWave;
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

// The deciding launch: 16 waves of a workgroup take a 16th of the line each, 64 positions at a time; the first kHeld
// steps stay in registers (lines of up to 8192 tokens are read once; with 32 steps, and five loops of
// as many copies, 24 lines of up to 500 tokens took 22 us instead of 11).  Three digits of 11, 11 and 10 bits: 2048 bins, two a
// thread.
constexpr int kSelectWaves = 16;
constexpr int kSelectThreads = kSelectWaves * kWave;
constexpr int kHeld = 8;
constexpr int kBins = 2 * kSelectThreads;

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictArgs a) {
  const EvictCall& c = a.c;
  const int64_t line = blockIdx.x;
  const int64_t head = line % c.kv_heads, row = line / c.kv_heads % c.batch, layer = line / c.kv_heads / c.batch;
  const int lane = lane_id(), wave = wave_in_block();
  __shared__ int32_t bad;
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t wave_of[kSelectWaves][2];
  __shared__ uint32_t digit_found, need_left;

  const int64_t said = int_at(c.lens, row, c.wide_lens), asked = int_at(c.keep, row, c.wide_keep);
  const int64_t len = said < 0 ? 0 : said, room = c.max_blocks * c.block_size;
  float* weights = c.weights + layer * c.weight_layer_stride + row * c.weight_row_stride + head * c.weight_head_stride;
  // A wave's positions: [seg * wave, seg * (wave + 1)), at most 2^29 in a line.
  const int32_t used = static_cast<int32_t>(len < room ? len : room);
  const int32_t seg = ((used + kSelectThreads - 1) / kSelectThreads) * kWave;
  const int32_t p0 = seg * wave + lane, steps = min(seg, max(used - seg * wave, 0) + kWave - 1) / kWave;
  const int32_t last = static_cast<int32_t>(used < c.weight_tokens ? used : c.weight_tokens);  // those with a weight
  auto weight_at = [&](int32_t p) {
    if (last == 0) return 0.0f;
    const float weight = weights[min(p, last - 1)];
    return p < last ? weight : 0.0f;
  };
  float held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = weight_at(p0 + i * kWave);
  // f(position, weight) for all steps of the wave, in order.
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (i < steps) f(p0 + i * kWave, held[i]);
    for (int32_t j = kHeld; j < steps; j += kHeld) {
      float more[kHeld];
#pragma unroll
      for (int i = 0; i < kHeld; ++i) more[i] = weight_at(p0 + (j + i) * kWave);
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (j + i < steps) f(p0 + (j + i) * kWave, more[i]);
    }
  };

  bool miss = asked < 0 || asked >= len || len > room;
  if (!miss) {
    for (int64_t p = threadIdx.x; p * c.block_size < len; p += kSelectThreads) {
      const int64_t blk = int_at(c.tables, row * c.table_stride + p, c.wide_tables);
      miss |= blk < 0 || blk >= c.num_blocks || (c.refs != nullptr && int_at(c.refs, blk, c.wide_refs) > 1);
    }
  }
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  if (miss) bad = 1;
  __syncthreads();
  const bool stays = bad != 0;
  if (threadIdx.x == 0) {
    *line_keep(a, line) = stays ? -1 : asked;
    if (layer == 0 && head == 0) c.kept[row] = stays ? len : asked;
  }
  if (stays) return;

  const int32_t keep = static_cast<int32_t>(asked);
  const int32_t first = static_cast<int32_t>(c.sinks < keep ? c.sinks : keep);
  const int32_t recent = static_cast<int32_t>(c.recent < keep - first ? c.recent : keep - first);
  const int32_t from = first, to = used - recent;  // where the heaviest are looked for

  // The key of the lightest one that stays, digit by digit from the top, and how many of that key stay.
  uint32_t key = 0, need = static_cast<uint32_t>(keep - first - recent);
  const bool choose = need > 0;
  int above_digit = 32;
  for (int shift : {21, 10, 0}) {
    if (!choose) break;
    const int width = above_digit - shift;
    bins[threadIdx.x] = bins[threadIdx.x + kSelectThreads] = 0;
    __syncthreads();
    each([&](int32_t p, float weight) {
      const uint32_t k = weight_key(weight);
      if (p >= from && p < to && (above_digit == 32 || k >> above_digit == key >> above_digit))
        atomicAdd(&bins[k >> shift & ((1u << width) - 1)], 1u);
    });
    __syncthreads();
    // Keys whose digit is at least that of the thread's two bins.
    const uint32_t low = bins[2 * threadIdx.x], high = bins[2 * threadIdx.x + 1];
    uint32_t upto = low + high;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint32_t y = __shfl_down(upto, o);
      if (lane + o < kWave) upto += y;
    }
    if (lane == 0) wave_of[wave][0] = upto;
    __syncthreads();
    for (int x = wave + 1; x < kSelectWaves; ++x) upto += wave_of[x][0];
    const uint32_t past_low = upto - low, past_high = past_low - high;
    if (past_low >= need && past_high < need) {
      digit_found = 2 * threadIdx.x + 1;
      need_left = need - past_high;
    } else if (upto >= need && past_low < need) {
      digit_found = 2 * threadIdx.x;
      need_left = need - past_low;
    }
    __syncthreads();
    key |= digit_found << shift;
    need = need_left;
    above_digit = shift;
  }

  // What stays: counted by each wave (lighter ones of the key itself only as far as they are needed, so both counts),
  // then marked, with the weights on their way to their places.
  auto kind = [&](int32_t p, float weight, uint64_t& sure, uint64_t& equal) {
    const uint32_t k = weight_key(weight);
    const bool between = choose && p >= from && p < to;
    equal = ballot(between && k == key);
    sure = ballot(p < used && (p < from || p >= to || (between && k > key)));
  };
  uint32_t sure_count = 0, equal_count = 0;
  each([&](int32_t p, float weight) {
    uint64_t sure, equal;
    kind(p, weight, sure, equal);
    sure_count += __popcll(sure);
    equal_count += __popcll(equal);
  });
  __syncthreads();
  if (lane == 0) {
    wave_of[wave][0] = sure_count;
    wave_of[wave][1] = equal_count;
  }
  __syncthreads();
  uint32_t rank = 0, same = 0;
  for (int x = 0; x < wave; ++x) {
    rank += wave_of[x][0];
    same += wave_of[x][1];
  }
  rank += min(same, need);
  uint64_t* bits = line_bits(a, line);
  float* moved = line_weights(a, line);
  const uint64_t lower = (uint64_t{1} << lane) - 1;
  each([&](int32_t p, float weight) {
    uint64_t sure, equal;
    kind(p, weight, sure, equal);
    const uint64_t mark = sure | ballot((equal >> lane & 1) != 0 && same + __popcll(equal & lower) < need);
    if (lane == 0) bits[p >> 6] = mark;
    if ((mark >> lane & 1) != 0) moved[rank + __popcll(mark & lower)] = weight;
    rank += __popcll(mark);
    same += __popcll(equal);
  });
  __syncthreads();
  for (int32_t p = threadIdx.x; p < last; p += kSelectThreads) weights[p] = p < keep ? moved[p] : 0.0f;
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
  for (int64_t word = 0; rank < keep && word < a.words; ++word) {
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

// ----- moving values of blocks whose rows are multiples of 16 bytes ------------------------------------
// A wave takes 16 bytes of a token's dims (or 8) and goes through a line's tokens 64 (128) at a time: 16 bytes a lane, whole
// pieces of the blocks' rows, kAhead steps on their way, the table entry of one more.  What stays is put behind one
// another in LDS, and leaves it as many tokens at a time as 16 bytes a lane again.  Bound by the read of every block that
// keeps a token (lines of 128 bytes hold the same 16 tokens of four dims, so single tokens are no cheaper to read).
constexpr int kAhead = 8;
// Bytes of LDS for a table row and a line's marks.  Where they need more, each step reads its own from memory, which
// waits for all loads that are on their way.
constexpr int64_t kMostStaged = 96 * 1024;

constexpr int64_t kFewWaves = 4096;  // of one of the two caches

struct MoveShape {
  int log_pieces;  // neighbouring lanes take this many pieces of 16 bytes of a block's row (log2)
  int log_block;   // log2(block_size), or -1
};

template <int ELT>
__device__ __forceinline__ typename VecType<ELT>::T element(const u32x4& v, int t) {
  if constexpr (ELT == 1) return static_cast<uint8_t>(elem8(v, t));
  else if constexpr (ELT == 2) return static_cast<uint16_t>(elem16(v, t));
  else return v[t];
}

// Half the dims of a wave, twice the tokens of a step.
template <int ELT, bool FEW>
constexpr int kDimsOf = (FEW ? 8 : 16) / ELT;

template <int ELT, bool FEW, bool STAGED, bool POW2>  // POW2: log_block is there
__global__ __launch_bounds__(kBlockThreads) void evict_move_kernel(const EvictArgs a, const MoveShape shape) {
  using T = typename VecType<ELT>::T;
  constexpr int kDims = kDimsOf<ELT, FEW>, kUnit = 16 / ELT;  // tokens of a lane
  constexpr int kTokens = FEW ? 2 * kWave : kWave, kWords = kTokens / kWave;
  constexpr int kPitch = 2 * kTokens + kUnit;  // tokens of a dim in LDS: less than a step's, and a step's more
  constexpr uint32_t kUnitBits = (1u << kUnit) - 1;
  const EvictCall& c = a.c;
  const int64_t line = blockIdx.x;
  const int kv = blockIdx.z, lane = lane_id(), wave = wave_in_block();
  __shared__ __attribute__((aligned(16))) T holds[kWavesPerBlock][kDims * kPitch + kUnit];
  extern __shared__ uint64_t marks[];  // the line's words, then the row's entries
  int32_t* entries = reinterpret_cast<int32_t*>(marks + a.words);
  const int64_t keep64 = uniform64(*line_keep(a, line));
  if (keep64 <= 0) return;
  const int32_t keep = static_cast<int32_t>(keep64), bs = static_cast<int32_t>(c.block_size);
  const int64_t head = line % c.kv_heads, row = line / c.kv_heads % c.batch, layer = line / c.kv_heads / c.batch;
  const int32_t len = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(int_at(c.lens, row, c.wide_lens)));
  const int32_t words = (len + kWave - 1) / kWave, steps = (len + kTokens - 1) / kTokens;
  const uint64_t* bits = line_bits(a, line);
  if constexpr (STAGED) {
    for (int64_t p = threadIdx.x; p * bs < len; p += kBlockThreads)
      entries[p] = static_cast<int32_t>(int_at(c.tables, row * c.table_stride + p, c.wide_tables));
    for (int32_t p = threadIdx.x; p < words; p += kBlockThreads) marks[p] = bits[p];
    __syncthreads();
  }
  const int32_t d0 = (blockIdx.y * kWavesPerBlock + wave) * kDims;
  if (d0 >= c.head_dim) return;
  // Lane: dim and unit of tokens, pieces of a row of a block next to each other.
  constexpr int kLogDims = __builtin_ctz(kDims);
  const int dim = lane >> shape.log_pieces & (kDims - 1);
  const int first = kUnit * ((lane & ((1 << shape.log_pieces) - 1)) |
                             (lane >> (shape.log_pieces + kLogDims) << shape.log_pieces));
  const bool mine = d0 + dim < c.head_dim;
  const uint8_t* plane = static_cast<const uint8_t*>(c.cache[kv]) + layer * c.cache_layer_stride[kv];
  const uint8_t* base = plane + (head * c.head_dim + min(d0 + dim, static_cast<int32_t>(c.head_dim) - 1)) * bs * ELT;
  const uint32_t block_bytes = static_cast<uint32_t>(c.cache_block_stride[kv]);
  auto column_of = [&](int32_t token) {
    return POW2 ? token >> shape.log_block : static_cast<int32_t>(static_cast<uint32_t>(token) / static_cast<uint32_t>(bs));
  };
  auto entry_of = [&](int32_t token) -> uint32_t {  // of a position below len
    if constexpr (STAGED) return entries[column_of(token)];
    else return static_cast<uint32_t>(row_block(c, row, token));
  };
  auto address = [&](uint32_t entry, int32_t token) {
    const int32_t place = POW2 ? token & (bs - 1) : token - column_of(token) * bs;
    return base + static_cast<uint64_t>(entry) * block_bytes + static_cast<uint64_t>(static_cast<uint32_t>(place)) * ELT;
  };
  auto mark_of = [&](int32_t word) {
    if constexpr (STAGED) return marks[min(word, words - 1)];
    else return bits[min(word, words - 1)];
  };

  T* hold = holds[wave];
  const uint32_t mine_hold = dim * kPitch;
  const uint32_t dump = kDims * kPitch;  // where the values go that do not stay
  const int bit0 = first % kWave, my_word = first / kWave;
  const uint64_t below = (uint64_t{1} << bit0) - 1;
  struct Marks {
    uint64_t of[kWords];
  };
  Marks mark_ahead[kAhead], next_mark;
  u32x4 ahead[kAhead];
#pragma unroll
  for (int k = 0; k < kWords; ++k) next_mark.of[k] = mark_of(k);
  uint32_t next_entry = entry_of(min(first, len - 1));
  auto mine_of = [&](const Marks& m) {
    uint64_t word = m.of[0];
#pragma unroll
    for (int k = 1; k < kWords; ++k) word = my_word == k ? m.of[k] : word;
    return word;
  };
  // Step `step` on its way, and the marks and entry of the one behind it.  Units that keep nothing read the beginning of
  // the layer, all lanes the same 16 bytes.
  auto issue = [&](int32_t step, Marks& mark, u32x4& values) {
#pragma unroll
    for (int k = 0; k < kWords; ++k)
      mark.of[k] = step * kWords + k < words ? static_cast<uint64_t>(uniform64(static_cast<int64_t>(next_mark.of[k]))) : 0;
    const bool some = (mine_of(mark) >> bit0 & kUnitBits) != 0;
    values = ld16_cached(some ? address(next_entry, step * kTokens + first) : plane);
#pragma unroll
    for (int k = 0; k < kWords; ++k) next_mark.of[k] = mark_of((step + 1) * kWords + k);
    next_entry = entry_of(min((step + 1) * kTokens + first, len - 1));
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) issue(i, mark_ahead[i], ahead[i]);
  int32_t level = 0, out = 0;  // tokens in LDS, and those that left it
  uint32_t out_entry = entry_of(min(first, len - 1));
  for (int32_t step0 = 0; out + level < keep && step0 < steps; step0 += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const Marks& mark = mark_ahead[i];
      uint64_t any = 0;
#pragma unroll
      for (int k = 0; k < kWords; ++k) any |= mark.of[k];
      if (any != 0) {
        const uint64_t my_mark = mine_of(mark);
        const uint32_t stay = static_cast<uint32_t>(my_mark >> bit0) & kUnitBits;
        uint32_t at = mine_hold + level + __popcll(my_mark & below);
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          if (k < my_word) at += __popcll(mark.of[k]);
          level += __popcll(mark.of[k]);
        }
#pragma unroll
        for (int t = 0; t < kUnit; ++t) {
          const uint32_t bit = stay >> t & 1u;
          hold[bit != 0 ? at : dump] = element<ELT>(ahead[i], t);
          at += bit;
        }
        __builtin_amdgcn_wave_barrier();
        if (level >= kTokens) {
          u32x4* from = reinterpret_cast<u32x4*>(hold + mine_hold + first);
          const u32x4 full = from[0], rest = from[kTokens / kUnit];
          if (mine) st16_cached(const_cast<uint8_t*>(address(out_entry, out + first)), full);
          from[0] = rest;
          out += kTokens;
          level -= kTokens;
          out_entry = entry_of(min(out + first, len - 1));
          __builtin_amdgcn_wave_barrier();
        }
      }
      issue(step0 + i + kAhead, mark_ahead[i], ahead[i]);
    }
  }
  const int32_t left = keep - out - first;  // of this lane's last unit
  if (mine && left > 0) {
    const T* from = hold + mine_hold + first;
    uint8_t* to = const_cast<uint8_t*>(address(out_entry, out + first));
    if (left >= kUnit) st16_cached(to, *reinterpret_cast<const u32x4*>(from));
    else
      for (int t = 0; t < left; ++t)
        reinterpret_cast<KVHIP_GLOBAL T*>(reinterpret_cast<uint64_t>(to))[t] = from[t];
  }
}

// Whether evict_move_kernel takes the caches, and how.
bool move_fits(const EvictCall& c, MoveShape& shape) {
  const int64_t unit = 16 / c.element_bytes;
  if (c.block_size % unit != 0) return false;
  for (int kv = 0; kv < 2; ++kv)
    if (((reinterpret_cast<uint64_t>(c.cache[kv]) | c.cache_layer_stride[kv] | c.cache_block_stride[kv]) & 15) != 0 ||
        c.cache_block_stride[kv] < 0 || c.cache_block_stride[kv] >= int64_t{1} << 32)
      return false;
  const int64_t pieces = c.block_size / unit;
  shape.log_pieces = pieces % 8 == 0 ? 3 : pieces == 4 ? 2 : pieces == 2 ? 1 : 0;
  shape.log_block = (c.block_size & (c.block_size - 1)) == 0 ? __builtin_ctzll(c.block_size) : -1;
  return true;
}

template <int ELT, bool FEW>
void launch_move(const EvictArgs& a, MoveShape shape, hipStream_t stream) {
  const EvictCall& c = a.c;
  constexpr int kLogUnits = __builtin_ctz(kWave / kDimsOf<ELT, FEW>);  // of a step
  if (shape.log_pieces > kLogUnits) shape.log_pieces = kLogUnits;
  constexpr int kSlice = kDimsOf<ELT, FEW> * kWavesPerBlock;
  const dim3 grid(a.lines, (c.head_dim + kSlice - 1) / kSlice, 2);
  const int64_t staged = a.words * 8 + c.max_blocks * 4;
  const bool pow2 = shape.log_block >= 0;
  if (staged > kMostStaged) {
    if (pow2) evict_move_kernel<ELT, FEW, false, true><<<grid, kBlockThreads, 0, stream>>>(a, shape);
    else evict_move_kernel<ELT, FEW, false, false><<<grid, kBlockThreads, 0, stream>>>(a, shape);
  } else {
    if (pow2) evict_move_kernel<ELT, FEW, true, true><<<grid, kBlockThreads, staged, stream>>>(a, shape);
    else evict_move_kernel<ELT, FEW, true, false><<<grid, kBlockThreads, staged, stream>>>(a, shape);
  }
}

template <int ELT>
void launch_moves(const EvictArgs& a, hipStream_t stream) {
  const EvictCall& c = a.c;
  MoveShape shape{};
  if (move_fits(c, shape)) {
    // Few waves: half the dims each, twice the tokens a step (40001 tokens of 16 lines, 16 bits: 119 us, against 186).
    // With many the longer pieces of memory are read a little faster (512 lines 279, against 295).
    const int64_t waves = a.lines * ((c.head_dim + kDimsOf<ELT, false> - 1) / kDimsOf<ELT, false>);
    if (waves < kFewWaves) launch_move<ELT, true>(a, shape, stream);
    else launch_move<ELT, false>(a, shape, stream);
    return;
  }
  const int64_t slices = (c.head_dim + kMoveDims * kWavesPerBlock - 1) / (kMoveDims * kWavesPerBlock);
  evict_move_any_kernel<ELT><<<dim3(a.lines, slices, 2), kBlockThreads, 0, stream>>>(a);
}

EvictArgs evict_args(const EvictCall& c) {
  EvictArgs a{};
  a.c = c;
  a.words = (c.max_blocks * c.block_size + kWave - 1) / kWave;
  a.lines = c.layers * c.batch * c.kv_heads;
  return a;
}

}  // namespace

int64_t evict_workspace(const EvictCall& c) {
  const EvictArgs a = evict_args(c);
  return a.lines * (8 + a.words * (8 + kWave * 4));
}

hipError_t launch_evict(const EvictCall& c, hipStream_t stream) {
  const EvictArgs a = evict_args(c);
  const int64_t lines = c.layers * c.batch * c.kv_heads;
  evict_select_kernel<<<dim3(lines), kSelectThreads, 0, stream>>>(a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  if (c.element_bytes == 1) launch_moves<1>(a, stream);
  else if (c.element_bytes == 2) launch_moves<2>(a, stream);
  else launch_moves<4>(a, stream);
  return hipGetLastError();
}

}  // namespace kvhip
