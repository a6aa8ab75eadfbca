// What the kernels over paged caches of plain values share: which positions a row tile and each of its rows see, and
// how a tile's positions are cut into parts.
#pragma once

#include "kv_attention.h"
#include "musa_aiter_kv_paged_attention.h"

namespace kvhip {

using CacheAttnCall = musa_aiter_hip_paged_attention_call;
using EvictCall = musa_aiter_hip_evict_call;

hipError_t launch_cache_attention(const CacheAttnCall& c, hipStream_t stream);
int64_t cache_attention_workspace(const CacheAttnCall& c);
hipError_t launch_attention_weights(const CacheAttnCall& c, hipStream_t stream);
hipError_t launch_evict(const EvictCall& c, hipStream_t stream);
int64_t evict_workspace(const EvictCall& c);

namespace catt {

using namespace attn;

struct CacheArgs {
  RowsArgs r;  // the call's rows, tables and lengths (scales, window and splits are not used)
  const int64_t* masks;
  int64_t mask_stride;
  float* weights;
  int64_t weight_row_stride, weight_head_stride;
  int32_t mask_words, weight_tokens;
  int32_t window, sinks;
  int32_t part, parts;   // positions of a part; the most parts that a line has
  int32_t slot_rows;     // rows of a part in the workspace
  int32_t tiles;         // row tiles of the launch
  int64_t lines;         // (row tile, kv head) pairs, or (row, head) pairs of the form for any shape
  float scale, factor;   // softmax_scale, and times log2(e)
  // What float32 takes from the two: scale + scale_rest is softmax_scale, lse_factor + lse_rest is factor / softmax_scale
  // (log2(e), with the rounding that factor has), so that (score * factor) - lse * (factor / scale) is small where
  // score * scale - lse is, however large the two are.
  float scale_rest, lse_factor, lse_rest;
};

// Weights are 2^(score - m), with m a row's maximum so far less kTop: fp16 ones keep their 11 bits down to 2^-28 of the
// largest.  The others have float32's range, and a weight of one for the maximum, so that products with its smallest
// values stay normal numbers; where sums with its largest ones pass its range, a row is done once more (see visit_row).
// Waves and parts hand on (m, l, o): the sum of the row's weights is l * 2^m, o what they make of the values.
template <int DT>
constexpr float kTop = DT == kLinF16 ? 14.0f : 0.0f;

// Positions that the rows of a tile see between them, as an axis without the gap between the first tokens and the
// window: place v is position v below `front`, v + gap from there on.  `front` and the window's begin are rounded to
// 16 positions, so that a unit of 8 places lies in one block.
struct View {
  int32_t before;          // position of the sequence's first row (a tree: the tokens in front of it)
  int32_t pos_lo, pos_hi;  // of the tile's first and last row
  int32_t begin, end;      // seen by any row, next to the first `first` positions
  int32_t first;
  int32_t front, gap, length;
};

__device__ __forceinline__ int32_t sequence_len(const CacheArgs& a, int32_t seq) {
  const int64_t said = seq_len(a.r.c, seq);
  return said < 0 ? 0 : said < kMostLen ? static_cast<int32_t>(said) : kMostLen;
}

// The view of rows [i_lo, i_hi] of a sequence of `count` rows.  At most 2^29 rows and positions of a table row, so
// that none of these sums leaves 32 bits; a sequence longer than kMostLen shows what one of that length does, since its
// rows lie past every position that a table row and a window reach.
__device__ __forceinline__ View make_view(const CacheArgs& a, int32_t seq, int32_t count, int32_t i_lo, int32_t i_hi) {
  View w;
  const int32_t len = sequence_len(a, seq);
  w.before = len - count;
  w.pos_lo = w.before + i_lo;
  w.pos_hi = w.before + i_hi;
  const int32_t upto = a.masks != nullptr ? len : w.pos_hi + 1;
  w.end = max(min(upto, a.r.room), 0);
  w.begin = a.window > 0 ? max(w.pos_lo - a.window + 1, 0) : 0;
  w.first = a.window > 0 ? min(a.sinks, w.end) : 0;
  const int32_t begin16 = w.begin & ~15;
  w.front = (w.first + 15) & ~15;
  if (w.front >= begin16) {
    w.front = w.gap = 0;
    w.length = w.end;
  } else {
    w.gap = begin16 - w.front;
    // A window past the end (a length past the table's room) leaves the first tokens, up to the end.
    w.length = w.end > begin16 ? w.front + w.end - begin16 : min(w.front, w.end);
  }
  return w;
}

__device__ __forceinline__ View tile_view(const CacheArgs& a, const RowTile& tile, int rows) {
  const int32_t last = min(tile.base + rows, tile.count * a.r.group) - 1;
  return make_view(a, tile.seq, tile.count, tile.base / a.r.group, last / a.r.group);
}

__device__ __forceinline__ int32_t position(const View& w, int32_t place) {
  return place < w.front ? place : place + w.gap;
}

// Bits of the n lowest of 8.
__device__ __forceinline__ uint32_t low_bits(int32_t n) { return (1u << min(max(n, 0), 8)) - 1u; }

// Which of the 8 positions from `token` on any row of the tile sees.
__device__ __forceinline__ uint32_t tile_bits(const View& w, int32_t token) {
  return low_bits(w.end - token) & (~low_bits(w.begin - token) | low_bits(w.first - token));
}

// What one row sees.
struct RowSight {
  int32_t pos;
  const int64_t* mask;  // a tree's row
};

__device__ __forceinline__ RowSight row_sight(const CacheArgs& a, const View& w, int32_t first_row, int32_t i) {
  return {w.before + i, a.masks != nullptr ? a.masks + (first_row + static_cast<int64_t>(i)) * a.mask_stride : nullptr};
}

// Which of the 8 positions from `token` on the row sees, where tile_bits has them.
__device__ __forceinline__ uint32_t row_bits(const CacheArgs& a, const View& w, const RowSight& row, int32_t token) {
  if (row.mask == nullptr) {
    uint32_t bits = low_bits(row.pos + 1 - token);
    if (a.window > 0) bits &= ~low_bits(row.pos - a.window + 1 - token) | low_bits(a.sinks - token);
    return bits;
  }
  const int32_t at = token - w.before;
  if (at <= -8) return 0xFFu;
  if (at < 0) return (low_bits(-at) | static_cast<uint32_t>(row.mask[0]) << -at) & 0xFFu;
  const int32_t word = at >> 6, bit = at & 63;
  uint64_t bits = word < a.mask_words ? static_cast<uint64_t>(row.mask[word]) >> bit : 0;
  if (bit > 56 && word + 1 < a.mask_words) bits |= static_cast<uint64_t>(row.mask[word + 1]) << (64 - bit);
  return static_cast<uint32_t>(bits) & 0xFFu;
}

// The block of a position below the view's end, or -1.
__device__ __forceinline__ int64_t position_block(const CacheArgs& a, int32_t seq, int32_t token) {
  const int64_t b = table_block(a.r.c, seq, static_cast<uint32_t>(token) / static_cast<uint32_t>(a.r.bs));
  return b >= 0 && b < a.r.num_blocks ? b : -1;
}

// Parts of a line whose view has `length` places, and the places of one of them.  Where `longest` of the call was too
// small, the last part takes what is left.
__device__ __forceinline__ int32_t part_count(const CacheArgs& a, int32_t length) {
  return max(min((length + a.part - 1) / a.part, a.parts), 1);
}
__device__ __forceinline__ Span part_places(const CacheArgs& a, int32_t length, int32_t s, int32_t count) {
  const int32_t lo = s * a.part;
  return {lo, s + 1 < count ? lo + a.part : length};
}

// Workspace: (m, l) of every part's rows, their outputs of head_dim values each (from a multiple of 16 bytes on: the
// matrix-core forms write 16 at a time), and a Line for each line.
struct Line {
  int32_t parts, first, count, base;  // parts 0: no rows
};

__host__ __device__ __forceinline__ int64_t ml_floats(int64_t slots) { return (2 * slots + 3) & ~int64_t{3}; }

__device__ __forceinline__ int64_t slot_row(const CacheArgs& a, int64_t line, int32_t s, int32_t row) {
  return (line * a.parts + s) * a.slot_rows + row;
}
__device__ __forceinline__ float* slot_ml(const CacheArgs& a, int64_t at) {
  return static_cast<float*>(a.r.c.workspace) + 2 * at;
}
__device__ __forceinline__ float* slot_out(const CacheArgs& a, int64_t at) {
  return static_cast<float*>(a.r.c.workspace) + ml_floats(a.lines * a.parts * a.slot_rows) + at * a.r.hd;
}
__device__ __forceinline__ Line* line_of(const CacheArgs& a, int64_t line) {
  return reinterpret_cast<Line*>(slot_out(a, a.lines * a.parts * a.slot_rows)) + line;
}

// ----- float32 throughout, one row: the form for any shape, and what a tile falls back to --------
constexpr int kVisitDims = 512;

// Scratch of a wave.
struct VisitScratch {
  float weight[kWave];
  int64_t place[kWave];
};

// One row's (m, l) and acc (dims lane + 64 i) over the places lo, lo + 1, .. of 64 at a time, `step` apart.  q: the
// row's query, in LDS.  l and acc are 2^-lower of what m says.  Sums over float32's largest values may be infinite with
// lower 0: a dim whose output is then no finite number is taken from a second visit with kLower, where such sums of up
// to 2^28 tokens are finite (and where the smallest values would be lost).
constexpr float kLower = 28.0f;

template <int DT, int DIMS>
__device__ __forceinline__ void visit_row(const CacheArgs& a, const View& w, int32_t seq, const RowSight& row,
                                          int32_t kv_head, const float* q, int32_t lo, int32_t hi, int32_t step,
                                          float lower, VisitScratch& scratch, float& m, float& l,
                                          float (&acc)[DIMS / kWave]) {
  const AttnCall& c = a.r.c;
  const int lane = lane_id();
  const int64_t bs = a.r.bs, hd = a.r.hd;
  constexpr int64_t kElt = DT == kLinF32 ? 4 : 2;
  m = -__builtin_inff();
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < DIMS / kWave; ++i) acc[i] = 0.0f;
  for (int32_t base = lo; base < hi; base += step) {
    const int32_t v = base + lane;
    float s = -__builtin_inff();
    int64_t off = -1;
    if (v < hi) {
      const int32_t token = position(w, v);
      const bool seen = (tile_bits(w, token) & row_bits(a, w, row, token) & 1u) != 0;
      const int64_t blk = seen ? position_block(a, seq, token) : -1;
      if (blk >= 0) {
        const int64_t in_block = kv_head * hd * bs + token % bs;
        const int64_t k = blk * (c.cache_block_stride[0] / kElt) + in_block;
        off = blk * (c.cache_block_stride[1] / kElt) + in_block;
        float dot = 0.0f;
        for (int64_t d = 0; d < hd; ++d) dot = __builtin_fmaf(q[d], load_q<DT>(c.cache[0], k + d * bs), dot);
        s = dot * a.factor;
      }
    }
    const float top = fmaxf(m, wave_max(s));
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    // A masked position's score is -inf; with a row's maximum of +inf its weight would be no number.
    const float p = off >= 0 ? __builtin_amdgcn_exp2f(s - ref - lower) : 0.0f;
    const float fade = __builtin_amdgcn_exp2f(m - ref);
    m = top;
    l = l * fade + wave_sum(p);
    scratch.weight[lane] = p;
    scratch.place[lane] = off;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < DIMS / kWave; ++i) {
      const int64_t d = lane + i * kWave;
      if (d >= hd) continue;
      float o = acc[i] * fade;
      for (int x = 0; x < kWave; ++x)
        if (scratch.place[x] >= 0)
          o = __builtin_fmaf(scratch.weight[x], load_q<DT>(c.cache[1], scratch.place[x] + d * bs), o);
      acc[i] = o;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// 2^(m - top), with m and top possibly both -inf.
__device__ __forceinline__ float fade_to(float m, float top) {
  return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - top);
}

__device__ __forceinline__ float log_sum(float m, float l) {
  return l == 0.0f ? -__builtin_inff() : (m + log2f(l)) * kLn2;
}

// Arguments of a launch in tiles of `size` rows (0: the form for any shape, a line per row and head).
CacheArgs cache_args(const CacheAttnCall& c, int size);
// Whether the caches' blocks can be read, and the output be written, as the matrix-core forms do.
bool tiles_fit(const CacheAttnCall& c);

}  // namespace catt
}  // namespace kvhip
