// What the attention kernels over block-scaled FP8 caches share: rows and their sequences, parts, the codes' way into
// matrix instructions, row tiles and table lookups.
#pragma once

#include "kv_serving.h"

namespace kvhip {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

using AttnCall = musa_aiter_hip_attention_call;

__device__ __forceinline__ int64_t int_at(const void* p, int64_t i, int wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// Rows [first, first + count) of sequence b; a row table that runs backwards or past the rows gives none.
struct SeqRows {
  int64_t first, count;
};

__device__ __forceinline__ SeqRows seq_rows(const AttnCall& c, int64_t b) {
  if (c.starts == nullptr) return {b, b < c.rows ? 1 : 0};
  const int64_t lo = int_at(c.starts, b, c.wide_starts), hi = int_at(c.starts, b + 1, c.wide_starts);
  if (lo < 0 || hi < lo || hi > c.rows) return {0, 0};
  return {lo, hi - lo};
}

// The sequence whose row t is, its first row and number of rows (seq -1: none); the same in all lanes.
struct RowSeq {
  int64_t seq, first, count;
};

__device__ __forceinline__ RowSeq row_sequence(const AttnCall& c, int64_t t) {
  if (c.starts == nullptr) return t < c.batch ? RowSeq{t, t, 1} : RowSeq{-1, 0, 0};
  for (int64_t b0 = 0; b0 < c.batch; b0 += kWave) {
    SeqRows r{0, 0};
    if (b0 + lane_id() < c.batch) r = seq_rows(c, b0 + lane_id());
    const uint64_t hit = ballot(t >= r.first && t < r.first + r.count);
    if (hit == 0) continue;
    const int src = __builtin_ctzll(hit);
    return {b0 + src, readlane64(r.first, src), readlane64(r.count, src)};
  }
  return {-1, 0, 0};
}

__device__ __forceinline__ int64_t seq_len(const AttnCall& c, int64_t b) { return int_at(c.lens, b, c.wide_lens); }

__device__ __forceinline__ int64_t table_block(const AttnCall& c, int64_t b, int64_t j) {
  return int_at(c.tables, b * c.table_stride + j, c.wide_tables);
}

// A query's 16-bit value, fp16 denormals included whatever the mode register says about them.
template <int DT>
__device__ __forceinline__ float query_value(uint16_t bits) {
  if constexpr (DT == kLinBF16) {
    return bf16_bits_to_f32(bits);
  } else {
    const uint32_t a = static_cast<uint32_t>(bits & 0x7FFFu) << 13;
    const uint32_t top = (bits & 0x7C00u) == 0x7C00u ? 0x7F800000u : 0u;  // infinities and NaN
    return __uint_as_float(__float_as_uint(__uint_as_float(a) * 0x1p112f) | top | static_cast<uint32_t>(bits & 0x8000u) << 16);
  }
}

template <int DT>
__device__ __forceinline__ float load_q(const void* base, int64_t i) {
  if constexpr (DT == kLinF32) return static_cast<const float*>(base)[i];
  else return lin_to_f32<DT>(static_cast<const uint16_t*>(base)[i]);
}

template <int DT>
__device__ __forceinline__ void store_o(void* base, int64_t i, float v) {
  if constexpr (DT == kLinF32) static_cast<float*>(base)[i] = v;
  else static_cast<uint16_t*>(base)[i] = static_cast<uint16_t>(f32_to_lin<DT>(v));
}

// Partial results in the workspace: (m, l) of `count` parts, then their acc of head_dim values each.  With splits
// > 1 part s of (row, head) rh is s * rows * heads + rh; with an even cut (splits 0) see FlowCut.
__device__ __forceinline__ float* part_ml(const AttnCall& c, int64_t part) {
  return static_cast<float*>(c.workspace) + 2 * part;
}
__device__ __forceinline__ float* part_acc(const AttnCall& c, int64_t count, int64_t part) {
  return static_cast<float*>(c.workspace) + 2 * count + part * c.head_dim;
}
// Behind them, for an even cut: the first and last workgroup of every line.
__device__ __forceinline__ uint32_t* line_owners(const AttnCall& c, int64_t count, int64_t line) {
  return static_cast<uint32_t*>(c.workspace) + (2 + c.head_dim) * count + 2 * line;
}

// A part begins at a multiple of a wave's 64 tokens and, but for the last one, holds whole turns of a workgroup's
// four waves.
constexpr int64_t kPartTokens = 64;
constexpr int64_t kTurnTokens = kPartTokens * kWavesPerBlock;

struct Span {
  int64_t lo, hi;
};

// Part s of the positions [lo, hi).
__device__ __forceinline__ Span part_span(int64_t lo, int64_t hi, int64_t s, int64_t splits) {
  lo = lo / kPartTokens * kPartTokens;
  if (hi <= lo) return {lo, lo};
  const int64_t turns = (hi - lo + kTurnTokens - 1) / kTurnTokens;
  const int64_t per = (turns + splits - 1) / splits * kTurnTokens;
  const int64_t from = lo + s * per;
  const int64_t to = from + per;
  return {from < hi ? from : hi, to < hi ? to : hi};
}

constexpr int kWaveTokens = 64;

using f32x4 = float __attribute__((ext_vector_type(4)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x2 = _Float16 __attribute__((ext_vector_type(2)));
using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using f32x2 = float __attribute__((ext_vector_type(2)));
using i16x2 = short __attribute__((ext_vector_type(2)));

template <int CODEC>
struct Mma;

template <>
struct Mma<kE4M3> {
  static constexpr int kCodeShift = 8;     // value = stored * 2^8
  static constexpr int kQueryTop = 14;     // query rows are scaled to [2^14, 2^15)
  static constexpr int kWeightTop = 14;    // probabilities times value scale to at most 2^14
  uint32_t one;                            // 1.0 twice, from behind the change of the mode register

  // fp16 denormals off: the products by `one` (v_pk_mul_f16) then flush what exponent-0 codes become.  None can
  // be moved in front of the change, which `one` comes out of, or be left out, as the compiler does not know it.
  // (The products are no inline asm: an asm result that a matrix instruction reads would miss its wait states.)
  __device__ __forceinline__ Mma() {
    asm volatile("s_setreg_imm32_b32 hwreg(HW_REG_MODE, 6, 2), 0\n\ts_nop 3\n\tv_mov_b32 %0, 0x3c003c00" : "=v"(one));
  }
  // Denormals on again.  The outputs' conversions stay behind it: f32_to_f16_bits holds a volatile asm too.
  __device__ __forceinline__ void done() const {
    asm volatile("s_setreg_imm32_b32 hwreg(HW_REG_MODE, 6, 2), 3\n\ts_nop 3" ::);
  }
  __device__ __forceinline__ uint32_t prepare(uint32_t w) const { return w; }
  // Two codes in the high bytes of the halves of w.
  __device__ __forceinline__ uint32_t pair(uint32_t w) const {
    const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, w) >> i16x2{1, 1}) & 0xBF80BF80u;
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, h) * __builtin_bit_cast(f16x2, one));
  }
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
  }
  static __device__ __forceinline__ f32x2 unpack(uint32_t v) {
    return __builtin_convertvector(__builtin_bit_cast(f16x2, v), f32x2);
  }
};

template <>
struct Mma<kE5M2> {
  static constexpr int kCodeShift = 112;
  static constexpr int kQueryTop = 100;
  static constexpr int kWeightTop = 40;
  __device__ __forceinline__ void done() const {}
  __device__ __forceinline__ uint32_t prepare(uint32_t w) const {  // zeros for exponent-0 codes
    const uint32_t m = ((w & 0x7C7C7C7Cu) + 0x7C7C7C7Cu) & 0x80808080u;
    return w & ((m - (m >> 7)) | 0x80808080u);
  }
  __device__ __forceinline__ uint32_t pair(uint32_t w) const {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, w) >> i16x2{3, 3}) & 0x8FE08FE0u;
  }
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
  }
  static __device__ __forceinline__ f32x2 unpack(uint32_t v) {
    return f32x2{__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)};
  }
};

// Summands that hold a query value and a probability (see above).
template <int CODEC, int DT>
constexpr int kQueryParts = CODEC == kE5M2 && DT == kLinF16 ? 2 : 1;
template <int CODEC, int DT>
constexpr int kWeightParts = CODEC == kE5M2 || DT == kLinF16 ? 2 : 1;

// Values that the compiler takes for new ones, so that what follows from them is computed (or read) again where it
// is written.  Held over the loops, the offsets of every load and the like take more registers than there are.
__device__ __forceinline__ int not_hoisted(int v) {  // uniform
  asm volatile("" : "+s"(v));
  return v;
}
__device__ __forceinline__ int reread(int v) {  // of the lanes
  asm volatile("" : "+v"(v));
  return v;
}
__device__ __forceinline__ int lane_now() { return reread(lane_id()); }

// Maximum and sum over the four lane groups of 16.
__device__ __forceinline__ float groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float groups_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Sizes as 32-bit numbers: rows * heads and the positions of a table row stay far below 2^31 (checked by the
// C entry), and registers are what this kernel has least of.
struct RowsArgs {
  AttnCall c;
  int32_t batch, heads, hd, bs, num_blocks, room;  // room: positions that a table row has place for
  int32_t group;        // heads per kv head
  int32_t block_shift;  // log2(block_size / 16), or -1
  int32_t seq_tiles;    // row tiles of every sequence (no row table)
  int32_t window, splits;
  int32_t slot_rows;  // even cut: rows of a part
};

// The reference m that weights are taken relative to is max(score + log2(value scale)), so that weight * value scale fits
// 16 bits.  Rounded to a score's steps that sum may lie half a step too low: below 2^25 (in base 2) by 1, a factor of 2 that
// there is place for, from there on by 2 and more.  Past kLiftedScores m is therefore the score itself; the weights are at
// most one then, and value scales up to 4 fit.
constexpr float kLiftedScores = 0x1p25f;

__device__ __forceinline__ float score_lift(float score, float value_scale) {
  const float lift = __builtin_amdgcn_fmed3f(__builtin_amdgcn_logf(value_scale), -100.0f, 100.0f);
  return fabsf(score) > kLiftedScores ? 0.0f : lift;
}

constexpr int32_t kMostRoom = 1 << 29;
// Lengths past it see what a row of kMostRoom positions would show them.
constexpr int32_t kMostLen = 3 << 29;

// The row tile of a workgroup: rows [first, first + count) of sequence `seq` from (position, head) row `base`.
struct RowTile {
  int32_t seq, first, count, base;
};

// Finds the `index`-th tile of `size` rows over all sequences (seq -1: past the last).
__device__ __forceinline__ RowTile find_tile(const RowsArgs& a, int32_t index, int size) {
  const AttnCall& c = a.c;
  if (c.starts == nullptr) {
    const int32_t seq = index / a.seq_tiles;
    if (seq >= a.batch) return {-1, 0, 0, 0};
    return {seq, seq, 1, (index - seq * a.seq_tiles) * size};
  }
  int32_t before = 0;
  for (int32_t b0 = 0; b0 < a.batch; b0 += kWave) {
    const int32_t b = b0 + lane_id();
    SeqRows r{0, 0};
    if (b < a.batch) r = seq_rows(c, b);
    const int32_t first = static_cast<int32_t>(r.first), count = static_cast<int32_t>(r.count);
    const int32_t tiles = (count * a.group + size - 1) / size;
    int32_t upto = tiles;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int32_t y = __shfl_up(upto, o);
      if (lane_id() >= o) upto += y;
    }
    const uint64_t hit = ballot(before + upto > index);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      const int32_t in_front = before + __builtin_amdgcn_readlane(upto - tiles, src);
      return {b0 + src, __builtin_amdgcn_readlane(first, src), __builtin_amdgcn_readlane(count, src),
              (index - in_front) * size};
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return {-1, 0, 0, 0};
}

// Whether rows that belong to no sequence are written: their outputs with fill_rows, their logarithms in every case (they
// are -inf, whoever brought the output).
__device__ __forceinline__ bool writes_loose_rows(const AttnCall& c) { return c.fill_rows || c.lse != nullptr; }

// Writes heads [head, head + heads) of this workgroup's share of those rows.  Its waves look at 64 rows together, at the
// sequences that have some of them (one row after the other took 45 us for 3800 rows in 21 tiles), and take turns at the
// rows that are left.
template <int DT>
__device__ __forceinline__ void fill_loose_rows(const AttnCall& c, int64_t worker, int64_t workers, int64_t head,
                                                int64_t heads) {
  const int lane = lane_id();
  for (int64_t t0 = worker * kWave; t0 < c.rows; t0 += workers * kWave) {
    bool owned = t0 + lane >= c.rows;
    for (int64_t b0 = 0; b0 < c.batch; b0 += kWave) {
      SeqRows r{0, 0};
      if (b0 + lane < c.batch) r = seq_rows(c, b0 + lane);
      uint64_t some = ballot(r.count > 0 && r.first < t0 + kWave && r.first + r.count > t0);
      for (; some != 0; some &= some - 1) {
        const int src = __builtin_ctzll(some);
        const int64_t first = readlane64(r.first, src), count = readlane64(r.count, src);
        owned |= t0 + lane >= first && t0 + lane < first + count;
      }
    }
    int turn = 0;
    for (uint64_t loose = ballot(!owned); loose != 0; loose &= loose - 1, ++turn) {
      if (turn % kWavesPerBlock != wave_in_block()) continue;
      const int64_t at = (t0 + __builtin_ctzll(loose)) * c.heads + head;
      if (c.fill_rows)
        for (int64_t d = lane; d < heads * c.head_dim; d += kWave) store_o<DT>(c.out, at * c.head_dim + d, 0.0f);
      if (c.lse != nullptr)
        for (int64_t h = lane; h < heads; h += kWave) c.lse[at + h] = -__builtin_inff();
    }
  }
}

// Table column of the 16-token group that begins at `token` (a multiple of 16).
__device__ __forceinline__ uint32_t group_column(const RowsArgs& a, int32_t token) {
  const uint32_t n16 = static_cast<uint32_t>(token) >> 4;
  return a.block_shift >= 0 ? n16 >> a.block_shift : n16 / (static_cast<uint32_t>(a.bs) >> 4);
}

// Its first token's place in the block.
__device__ __forceinline__ int32_t group_place(const RowsArgs& a, int32_t token) {
  return token - static_cast<int32_t>(group_column(a, token)) * a.bs;
}

__device__ __forceinline__ uint32_t load4(const uint8_t* p) {
  return *reinterpret_cast<const KVHIP_GLOBAL uint32_t*>(reinterpret_cast<uint64_t>(p));
}

// The table entry of a group, on its way: nothing is done with it where it is loaded, which would wait for it and for
// the codes that were asked for before it.
struct Entry {
  uint32_t lo, hi;
  bool inside;  // the group has tokens that are seen, or are only masked next to some
};

__device__ __forceinline__ Entry load_entry(const RowsArgs& a, const uint8_t* row, int32_t token, int32_t end) {
  const uint32_t column = group_column(a, min(token, end - 1));
  const uint8_t* p = row + static_cast<uint64_t>(column) * (a.c.wide_tables ? 8 : 4);
  return {load4(p), load4(p + (a.c.wide_tables ? 4 : 0)), token < end};
}

// The same in the first tile of a part, which is rounded down to whole tiles: groups that end at or in front of `begin`,
// where the window of the first row does, are not taken.  Their pages may be anybody's by then, and a scale that is no
// number there would go through its weight of zero into the sums.
__device__ __forceinline__ Entry load_first_entry(const RowsArgs& a, const uint8_t* row, int32_t token, int32_t begin,
                                                  int32_t end) {
  Entry e = load_entry(a, row, token, end);
  e.inside = e.inside && token + 16 > begin;
  return e;
}

// Its block, or -1.
__device__ __forceinline__ int32_t entry_block(const RowsArgs& a, const Entry& e) {
  const bool good = e.inside && e.lo < static_cast<uint32_t>(a.num_blocks) && (!a.c.wide_tables || e.hi == 0);
  return good ? static_cast<int32_t>(e.lo) : -1;
}

// Positions [lo, hi) that a row sees.
struct Sight {
  int32_t lo, hi;
};

// Positions that the rows of a tile see between them.
struct Reach {
  int32_t before;           // position of the sequence's first row
  int32_t pos_lo, pos_hi;   // of the tile's first and last row
  int32_t begin, end;       // seen by any row
};

__device__ __forceinline__ Reach tile_reach(const RowsArgs& a, const RowTile& tile, int rows) {
  const int64_t said = seq_len(a.c, tile.seq);
  const int32_t len = said < 0 ? 0 : said < kMostLen ? static_cast<int32_t>(said) : kMostLen;
  Reach r;
  r.before = len - tile.count;
  r.pos_lo = r.before + tile.base / a.group;
  r.pos_hi = r.before + (min(tile.base + rows, tile.count * a.group) - 1) / a.group;
  r.end = min(r.pos_hi + 1, a.room);
  r.begin = a.window > 0 ? max(r.pos_lo - a.window + 1, 0) : 0;
  return r;
}

// Row tiles of `size` that the sequences of a call can have together.
inline int64_t tiles_bound(const AttnCall& c, int size) {
  const int64_t group = c.heads / c.kv_heads;
  if (c.starts == nullptr) return c.batch * ((group + size - 1) / size);
  return c.rows * group / size + c.batch;
}

inline RowsArgs rows_args(const AttnCall& c, int size) {
  RowsArgs a{};
  a.c = c;
  a.batch = static_cast<int32_t>(c.batch);
  a.heads = static_cast<int32_t>(c.heads);
  a.hd = static_cast<int32_t>(c.head_dim);
  a.bs = static_cast<int32_t>(c.block_size);
  a.num_blocks = static_cast<int32_t>(c.num_blocks);
  a.room = static_cast<int32_t>(c.max_blocks * c.block_size);
  a.window = static_cast<int32_t>(c.window < kMostRoom ? c.window : kMostRoom);
  a.splits = static_cast<int32_t>(c.splits);
  a.group = static_cast<int32_t>(c.heads / c.kv_heads);
  const int64_t b16 = c.block_size / 16;
  a.block_shift = (b16 & (b16 - 1)) == 0 ? __builtin_ctzll(b16) : -1;
  a.seq_tiles = (a.group + size - 1) / size;
  return a;
}

// kv_attention_wide.hip: a call with a row table, in tiles of kWideRows rows.
constexpr int kWideRows = 128;
hipError_t launch_wide(const AttnCall& c, hipStream_t stream);

}  // namespace attn
}  // namespace kvhip
