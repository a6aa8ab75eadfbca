// Attention over a paged FP8 cache with one scale per (block, head): kv_paged_attention_fp8.
//
//   s_j = softmax_scale * ks[blk(j), h] * sum_d q_d decode(K[blk(j), h, d, j % bs])
//   o_d = sum_j e^(s_j - lse) vs[blk(j), h] decode(V[blk(j), h, d, j % bs]),  lse = log sum_j e^(s_j)
//
// over the positions j that the row sees.  One pass over the cache with a running maximum and sum in base 2
// (p_j = 2^(s_j log2(e) - m)); parts of a sequence that run side by side leave (m, l, acc) in a workspace and
// a second launch joins them.
#include "kv_attention.h"

namespace kvhip {
namespace {

using namespace attn;

// ----- any shape and type: one workgroup per (row, head, part), fp32 throughout -------------------
constexpr int kAnyMaxDim = 512;

template <int DT, int CODEC>
__global__ __launch_bounds__(kBlockThreads) void attention_any_kernel(const AttnCall c) {
  const int64_t t = blockIdx.x, hq = blockIdx.y, split = blockIdx.z;
  const int64_t rh = t * c.heads + hq;
  __shared__ float q[kAnyMaxDim];
  __shared__ float weight[kWavesPerBlock][kWave];
  __shared__ int64_t place[kWavesPerBlock][kWave];
  __shared__ float acc_of[kWavesPerBlock][kAnyMaxDim];
  __shared__ float m_of[kWavesPerBlock], l_of[kWavesPerBlock];
  const int lane = lane_id(), wave = wave_in_block();
  const int64_t bs = c.block_size;

  const RowSeq row = row_sequence(c, t);
  const int64_t seq = row.seq;
  if (seq < 0) {
    if (split != 0) return;
    if (c.fill_rows)
      for (int64_t d = threadIdx.x; d < c.head_dim; d += kBlockThreads) store_o<DT>(c.out, rh * c.head_dim + d, 0.0f);
    if (c.lse != nullptr && threadIdx.x == 0) c.lse[rh] = -__builtin_inff();
    return;
  }
  const int64_t pos = seq_len(c, seq) - row.count + (t - row.first);
  const int64_t group = c.heads / c.kv_heads, head = hq / group;
  for (int64_t d = threadIdx.x; d < c.head_dim; d += kBlockThreads)
    q[d] = load_q<DT>(c.query, t * c.query_row_stride + hq * c.query_head_stride + d);
  __syncthreads();
  int64_t hi = pos + 1;
  if (hi > c.max_blocks * bs) hi = c.max_blocks * bs;
  const int64_t lo = c.window > 0 && pos >= c.window ? pos - c.window + 1 : 0;
  const Span span = part_span(lo, hi, split, c.splits);

  float m = -__builtin_inff(), l = 0.0f;
  float acc[kAnyMaxDim / kWave] = {};
  const float factor = static_cast<float>(c.softmax_scale) * kLog2e;
  for (int64_t base = span.lo + wave * kWave; base < span.hi; base += kBlockThreads) {
    const int64_t j = base + lane;
    float s = -__builtin_inff();
    int64_t off = -1;
    float vs = 0.0f;
    if (j < span.hi && j >= lo) {
      const int64_t blk = table_block(c, seq, j / bs);
      if (blk >= 0 && blk < c.num_blocks) {
        const uint8_t* k = static_cast<const uint8_t*>(c.cache[0]) + blk * c.cache_block_stride[0] +
                           head * c.head_dim * bs + j % bs;
        float dot = 0.0f;
        for (int64_t d = 0; d < c.head_dim; ++d) dot = __builtin_fmaf(q[d], fp8_decode<CODEC>(k[d * bs]), dot);
        s = dot * (c.scale[0][blk * c.scale_block_stride[0] + head * c.scale_head_stride[0]] * factor);
        vs = c.scale[1][blk * c.scale_block_stride[1] + head * c.scale_head_stride[1]];
        off = blk * c.cache_block_stride[1] + head * c.head_dim * bs + j % bs;
      }
    }
    const float top = fmaxf(m, wave_max(s));
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    const float p = __builtin_amdgcn_exp2f(s - ref), fade = __builtin_amdgcn_exp2f(m - ref);
    m = top;
    l = l * fade + wave_sum(p);
    weight[wave][lane] = off >= 0 ? p * vs : 0.0f;
    place[wave][lane] = off;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < kAnyMaxDim / kWave; ++i) {
      const int64_t d = lane + i * kWave;
      if (d >= c.head_dim) continue;
      float o = acc[i] * fade;
      for (int x = 0; x < kWave; ++x)
        if (place[wave][x] >= 0)
          o = __builtin_fmaf(weight[wave][x],
                             fp8_decode<CODEC>(static_cast<const uint8_t*>(c.cache[1])[place[wave][x] + d * bs]), o);
      acc[i] = o;
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (lane == 0) {
    m_of[wave] = m;
    l_of[wave] = l;
  }
#pragma unroll
  for (int i = 0; i < kAnyMaxDim / kWave; ++i)
    if (lane + i * kWave < c.head_dim) acc_of[wave][lane + i * kWave] = acc[i];
  __syncthreads();
  float top = m_of[0];
  for (int w = 1; w < kWavesPerBlock; ++w) top = fmaxf(top, m_of[w]);
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  float fade[kWavesPerBlock], sum = 0.0f;
  for (int w = 0; w < kWavesPerBlock; ++w) {
    fade[w] = __builtin_amdgcn_exp2f(m_of[w] - ref);
    sum += l_of[w] * fade[w];
  }
  for (int64_t d = threadIdx.x; d < c.head_dim; d += kBlockThreads) {
    float o = 0.0f;
    for (int w = 0; w < kWavesPerBlock; ++w) o += acc_of[w][d] * fade[w];
    if (c.splits > 1) {
      if (sum != 0.0f) part_acc(c, c.splits * c.rows * c.heads, split * c.rows * c.heads + rh)[d] = o;
      continue;
    }
    store_o<DT>(c.out, rh * c.head_dim + d, sum == 0.0f ? 0.0f : o / sum);
  }
  if (threadIdx.x == 0) {
    if (c.splits > 1) {
      part_ml(c, split * c.rows * c.heads + rh)[0] = top;
      part_ml(c, split * c.rows * c.heads + rh)[1] = sum;
    } else if (c.lse != nullptr) {
      c.lse[rh] = sum == 0.0f ? -__builtin_inff() : (top + log2f(sum)) * kLn2;
    }
  }
}

// ----- matrix-core form ---------------------------------------------------------------------------
// A wave takes 64 cached tokens and 16 * NT query rows (row = position and head within the kv head's group) at
// a time: S^T = K Q^T, then O^T += V^T P^T, with 16x16x32 matrix instructions.  Everything stays in the lane
// that loaded it.  With x = lane % 16 and g = lane / 16:
//   * K: lane (x, g) loads the 4 tokens 16 (x / 4) + 4 (x % 4) .. + 3 of rows d = 4 l + g (one dword each: 16
//     lanes and 4 rows make 64-byte runs).  Byte i of the dwords of 8 rows is the A operand of the product for
//     tokens {4 x + i}, so four products (i = 0..3) cover the 64 tokens.
//   * Their results give lane (x, g) the scores of query row x with tokens 16 g + 4 r + i: the 16 tokens of one
//     group, which lie in one block (block sizes are multiples of 16), so scales and masks are per lane.
//   * V: lane (x, g) loads the 16 tokens of group g for d = 16 l + x (16 bytes).  Its bytes and the lane's
//     probabilities are the operands of V^T P^T in the same token order: no value crosses lanes but the
//     running maximum.
// Codes become 16-bit floats by shifts: E4M3 as fp16 with the value times 2^-8 (sign, 4 exponent and 3 mantissa
// bits fall on fp16's fields; the all-ones code is the ordinary 480 * 2^-8), E5M2 as bf16 times 2^-112.  Codes of
// exponent 0 are zeros: for fp16 a multiplication by one flushes them, with the mode register's fp16 denormals
// off; for bf16 their bits are masked.  Query rows are scaled by a power of two so that 16 bits hold them (two
// summands of bf16 hold an fp16 query); next to E4M3 codes what is 2^-28 of a row's largest and less becomes zero there,
// as the weights below it do.  Probabilities times value scale are rounded to 11 bits (8 + 8 bits in
// two bf16 summands, 11 + 11 in two fp16 summands where the output is fp16 and one rounding would show).
// The value scale of a block enters the running maximum, m = max(s_j + log2 vs_j), so that the weights fit fp16
// whatever the scales are (see score_lift); l = sum 2^(s_j - m) needs no such care in fp32.
// Memory bounds long decode steps: 64 rows of 295 to 8192 tokens (254565 in all; 32 heads, 8 kv heads, 128 dims) 116 us,
// 4.5 TB/s (a large copy 4.7), two rows of 131000 and 108683 tokens 106 us, 4.6 TB/s.  Short ones are a chain of dependent
// loads: 4 rows of up to 500 tokens 11 us.
// Query rows as B operands, in LDS (in registers they would cost every wave 16 for 128 dims and a third wave per
// SIMD its place): element j of step s of lane (x, g) is d = 32 s + 4 j + g of row x.
template <int HDP, int NT, int CODEC, int DT>
struct QueryTiles {
  u32x4 q[NT][kQueryParts<CODEC, DT>][HDP / 32][kWave];
  float factor[NT][16];  // scores times this (and the key scale) are in base 2

  // Rows of tile n by one wave; `row` is readable, and without `mine` the row is zeros.
  template <bool EXACT>
  __device__ __forceinline__ void fill(const RowsArgs& a, int n, const uint16_t* row, bool mine) {
    const int lane = lane_now(), x = lane & 15, g = lane >> 4;
    float most = 0.0f;
    uint16_t raw[HDP / 4];
#pragma unroll
    for (int l = 0; l < HDP / 4; ++l) {
      const int d = 4 * l + g;
      raw[l] = row[EXACT ? d : min(d, a.hd - 1)];
      if (!mine || (!EXACT && d >= a.hd)) raw[l] = 0;
    }
#pragma unroll
    for (int l = 0; l < HDP / 4; ++l) most = fmaxf(most, fabsf(query_value<DT>(raw[l])));
    most = groups_max(most);
    const bool fine = most > 0.0f && most < __builtin_inff();
    const int up = fine ? Mma<CODEC>::kQueryTop - ilogbf(most) : 0;
    if (g == 0)
      factor[n][x] = __builtin_ldexpf(static_cast<float>(a.c.softmax_scale) * kLog2e, Mma<CODEC>::kCodeShift - up);
#pragma unroll
    for (int s = 0; s < HDP / 32; ++s) {
      u32x4 v[kQueryParts<CODEC, DT>];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        float lo = __builtin_ldexpf(query_value<DT>(raw[8 * s + j]), up);
        float hi = __builtin_ldexpf(query_value<DT>(raw[8 * s + j + 1]), up);
#pragma unroll
        for (int part = 0; part < kQueryParts<CODEC, DT>; ++part) {
          v[part][j / 2] = Mma<CODEC>::pack(lo, hi);
          const f32x2 took = Mma<CODEC>::unpack(v[part][j / 2]);
          lo -= took[0];
          hi -= took[1];
        }
      }
#pragma unroll
      for (int part = 0; part < kQueryParts<CODEC, DT>; ++part) q[n][part][s][lane] = v[part];
    }
  }
};

struct GroupIds {
  int32_t k, v;  // blocks of the groups whose keys and values the lane loads
};

struct GroupEntries {
  Entry k, v;
};

__device__ __forceinline__ GroupEntries load_entries(const RowsArgs& a, const uint8_t* row, int32_t token, int32_t end) {
  const int lane = lane_now(), x = lane & 15, g = lane >> 4;
  return {load_entry(a, row, token + 16 * (x >> 2), end), load_entry(a, row, token + 16 * g, end)};
}

__device__ __forceinline__ GroupEntries load_first_entries(const RowsArgs& a, const uint8_t* row, int32_t token,
                                                           int32_t begin, int32_t end) {
  const int lane = lane_now(), x = lane & 15, g = lane >> 4;
  return {load_first_entry(a, row, token + 16 * (x >> 2), begin, end),
          load_first_entry(a, row, token + 16 * g, begin, end)};
}

__device__ __forceinline__ GroupIds group_ids(const RowsArgs& a, const GroupEntries& e) {
  return {entry_block(a, e.k), entry_block(a, e.v)};
}

// DIMS rows of the keys of 64 tokens: dword l is row d = first + 4 l + g of the lane's 4 tokens.  A group without a block reads block
// 0, which every cache has; its scores are masked.  Without EXACT rows past head_dim read the last one: the
// query is zero there.
template <int DIMS, bool EXACT>
__device__ __forceinline__ void load_keys(const RowsArgs& a, int64_t head_off, int32_t token, const GroupIds& ids,
                                          int first, uint32_t* k) {
  const AttnCall& c = a.c;
  const int lane = lane_now(), x = lane & 15, g = lane >> 4;
  const int32_t bs = a.bs;
  const uint8_t* p = static_cast<const uint8_t*>(c.cache[0]) + static_cast<int64_t>(ids.k < 0 ? 0 : ids.k) *
                     c.cache_block_stride[0] + head_off + group_place(a, token + 16 * (x >> 2)) + 4 * (x & 3);
  if constexpr (EXACT) {
    p += (first + g) * bs;
#pragma unroll
    for (int l = 0; l < DIMS / 4; ++l, p += 4 * bs) k[l] = load4(p);
  } else {
    const int last = a.hd - 1, step = not_hoisted(bs);
#pragma unroll
    for (int l = 0; l < DIMS / 4; ++l) k[l] = load4(p + min(first + 4 * l + g, last) * step);
  }
}

// Scales of the lane's group g.
struct GroupScales {
  float ks, vs;
  bool seen;  // the group has a block in the cache
};

__device__ __forceinline__ GroupScales load_scales(const AttnCall& c, int32_t head, const GroupIds& ids) {
  const int64_t blk = ids.v < 0 ? 0 : ids.v;
  return {c.scale[0][blk * c.scale_block_stride[0] + head * c.scale_head_stride[0]],
          c.scale[1][blk * c.scale_block_stride[1] + head * c.scale_head_stride[1]], ids.v >= 0};
}

// DIMS rows of the values of 64 tokens: piece l is row d = first + 16 l + x of the 16 tokens of group g (rows past
// head_dim as above: outputs past it are not stored).
template <int DIMS, bool EXACT>
__device__ __forceinline__ void load_values(const RowsArgs& a, int64_t head_off, int32_t token, const GroupIds& ids,
                                            int first, u32x4* v) {
  const AttnCall& c = a.c;
  const int lane = lane_now(), x = lane & 15;
  const int32_t bs = a.bs;
  const int64_t blk = ids.v < 0 ? 0 : ids.v;
  const uint8_t* p = static_cast<const uint8_t*>(c.cache[1]) + blk * c.cache_block_stride[1] + head_off +
                     group_place(a, token + 16 * (lane >> 4));
  if constexpr (EXACT) {
    p += (first + x) * bs;
#pragma unroll
    for (int l = 0; l < DIMS / 16; ++l, p += 16 * bs) v[l] = ld16_cached(p);
  } else {
    const int last = a.hd - 1, step = not_hoisted(bs);
#pragma unroll
    for (int l = 0; l < DIMS / 16; ++l) v[l] = ld16_cached(p + min(first + 16 * l + x, last) * step);
  }
}

// Running state of 16 query rows: lane (x, g) holds row x, dims 16 l + 4 g + r, and its own tokens' share of l.
template <int HDP>
struct RowState {
  f32x4 acc[HDP / 16];
  float m, l;
};

// Adds DIMS dims' part, from step FIRST on, of the scores of 16 * NT rows with 64 tokens, before scaling: element r
// of product i is token 16 g + 4 r + i.
template <int FIRST, int DIMS, int HDP, int NT, int CODEC, int DT>
__device__ __forceinline__ void key_products(const Mma<CODEC>& mma, const uint32_t* k,
                                             const QueryTiles<HDP, NT, CODEC, DT>& queries, f32x4 (*score)[4]) {
  const int lane = lane_now();
#pragma unroll
  for (int step = 0; step < DIMS / 32; ++step) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = mma.prepare(k[8 * step + j]);
    u32x4 q[NT][kQueryParts<CODEC, DT>];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int part = 0; part < kQueryParts<CODEC, DT>; ++part) q[n][part] = queries.q[n][part][FIRST + step][lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 a;
      // Bytes i of rows j and j + 1 into the high bytes of the halves.
      const uint32_t sel = 0x000C000Cu | (static_cast<uint32_t>(i) << 8) | (static_cast<uint32_t>(4 + i) << 24);
#pragma unroll
      for (int j = 0; j < 8; j += 2) a[j / 2] = mma.pair(__builtin_amdgcn_perm(w[j + 1], w[j], sel));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int part = 0; part < kQueryParts<CODEC, DT>; ++part)
          score[n][i] = Mma<CODEC>::mma(a, q[n][part], score[n][i]);
    }
  }
}

// One step of the running softmax: scores in, weights (probability * value scale) out; rescales the state where
// the maximum grew.
template <int HDP, int CODEC, typename SightOf>
__device__ __forceinline__ void soften(f32x4* score, float factor, const GroupScales& scales, bool masked,
                                       int32_t token, SightOf sight_of, RowState<HDP>& s) {
  const float f = factor * scales.ks, vs = scales.vs;
  const bool seen = scales.seen;
#pragma unroll
  for (int i = 0; i < 4; ++i) score[i] *= f;
  if (masked) {
    const int first = token + 16 * (lane_now() >> 4);
    const Sight sight = sight_of();
    const int lo = sight.lo - first, hi = seen ? sight.hi - first : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (4 * r + i < lo || 4 * r + i >= hi) score[i][r] = -__builtin_inff();
  }
  float most = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) most = fmaxf(most, score[i][r]);
  const float top = fmaxf(s.m, groups_max(most + score_lift(most, vs)));
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  if (ballot(top > s.m) != 0) {
    const float fade = __builtin_amdgcn_exp2f(s.m - ref);
    s.l *= fade;
#pragma unroll
    for (int l = 0; l < HDP / 16; ++l) s.acc[l] *= fade;
    s.m = top;
  }
  const float weight = seen ? __builtin_ldexpf(vs, Mma<CODEC>::kWeightTop) : 0.0f;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float p = __builtin_amdgcn_exp2f(score[i][r] - ref);
      sum += p;
      score[i][r] = p * weight;
    }
  s.l += sum;
}

// Weights as B operands of step `step`: tokens (0, 2), (1, 3) of the group's dword 2 step, then of the next one.
template <int CODEC, int DT>
__device__ __forceinline__ void pack_weights(const f32x4* score, int step, u32x4* p) {
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const int r = 2 * step + (h >> 1), i = h & 1;
    float a = score[i][r], b = score[i + 2][r];
#pragma unroll
    for (int part = 0; part < kWeightParts<CODEC, DT>; ++part) {
      p[part][h] = Mma<CODEC>::pack(a, b);
      const f32x2 took = Mma<CODEC>::unpack(p[part][h]);
      a -= took[0];
      b -= took[1];
    }
  }
}

// Adds weights times values to the state's dims from 16 * FIRST on.
template <int FIRST, int DIMS, int HDP, int NT, int CODEC, int DT>
__device__ __forceinline__ void value_products(const Mma<CODEC>& mma, const u32x4* v,
                                               u32x4 (*p)[2][kWeightParts<CODEC, DT>], RowState<HDP>* state) {
#pragma unroll
  for (int step = 0; step < 2; ++step) {
#pragma unroll
    for (int l = 0; l < DIMS / 16; ++l) {
      u32x4 a;
#pragma unroll
      for (int h = 0; h < 4; h += 2) {
        const uint32_t w = mma.prepare(v[l][2 * step + (h >> 1)]);
        a[h] = mma.pair(w << 8);
        a[h + 1] = mma.pair(w);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int part = 0; part < kWeightParts<CODEC, DT>; ++part)
          state[n].acc[FIRST + l] = Mma<CODEC>::mma(a, p[n][step][part], state[n].acc[FIRST + l]);
    }
  }
}

// One workgroup per (row tile, kv head, part): its four waves take turns at the part's 64-token tiles and join
// what they have in LDS, 128 dims at a time.  A wave loads the next tile's keys once this tile's are used up and
// its values behind this tile's, so either the one or the other is on its way all the time.
constexpr int kJoinDims = 128;

// Waves per SIMD that the registers of a variant leave room for (without spills; looked up in the compiler's report).
constexpr int rows_occupancy(int hdp, bool exact, int tiles, int codec) {
  if (hdp * tiles > 128) return 1;
  return tiles > 1 || (hdp == 128 && !exact && codec == kE5M2) ? 2 : 3;
}
constexpr int kJoinStride = kJoinDims + 4;

// A row tile's work on cached tokens [lo, hi), and where its result goes: the output (parts 0), or the `parts` of
// the workspace, row r of the tile to part first_part + r or, with by_row, first_part + its (row, head) number.
struct Segment {
  RowTile tile;
  int32_t head, lo, hi;
  int64_t parts, first_part;
  bool by_row;
};

// What row r of a tile sees.  (Worked out where a tile of tokens needs it: held, it would cost registers.)
__device__ __forceinline__ Sight row_sight(const RowsArgs& a, const RowTile& tile, int32_t before, int32_t r) {
  const int32_t at = tile.base + r, pos = before + at / a.group;
  if (at >= tile.count * a.group) return {0, 0};
  return {a.window > 0 ? max(pos - a.window + 1, 0) : 0, min(pos + 1, a.room)};
}

template <int HDP, int NT, int CODEC, int DT>
struct RowsShared {
  QueryTiles<HDP, NT, CODEC, DT> queries;
  float joined[kWavesPerBlock][16][kJoinStride];
  float ml[kWavesPerBlock][16][2];
};

template <int HDP, bool EXACT, int NT, int CODEC, int DT>
__device__ __forceinline__ void run_segment(const RowsArgs& a, const Segment& seg, const Reach& reach,
                                            RowsShared<HDP, NT, CODEC, DT>& shared) {
  const AttnCall& c = a.c;
  const RowTile& tile = seg.tile;
  const int32_t head = seg.head, group = a.group, in_seq = tile.count * group, before = reach.before;
  const int lane = lane_now(), x = lane & 15, wave = wave_in_block();
  // Tiles of tokens inside [all_lo, all_hi) are seen whole by every row.
  const int32_t all_lo = a.window > 0 ? max(reach.pos_hi - a.window + 1, 0) : 0;
  const int32_t last = seg.hi, all_hi = min(reach.pos_lo + 1, last);
  const int64_t head_off = static_cast<int64_t>(head) * a.hd * a.bs;
  const uint8_t* row = static_cast<const uint8_t*>(c.tables) +
                       tile.seq * c.table_stride * (c.wide_tables ? 8 : 4);

  constexpr int32_t kStep = kWavesPerBlock * kWaveTokens;
  // 256 dims go in two halves through the same registers.
  constexpr int kDims = HDP <= 128 ? HDP : HDP / 2;
  int32_t token = seg.lo + wave * kWaveTokens;
  uint32_t k[kDims / 4];
  u32x4 v[kDims / 16];
  GroupIds ids;
  GroupEntries next_entries;
  GroupScales scales;
  if (token < last) {  // on their way while the queries are read
    const GroupEntries entries = load_first_entries(a, row, token, reach.begin, last);
    next_entries = load_entries(a, row, token + kStep, last);
    ids = group_ids(a, entries);
    scales = load_scales(c, head, ids);
    load_keys<kDims, EXACT>(a, head_off, token, ids, 0, k);
    load_values<kDims, EXACT>(a, head_off, token, ids, 0, v);
  }

  const Mma<CODEC> mma;
  // Rows and what they see; the waves share the queries.
  QueryTiles<HDP, NT, CODEC, DT>& queries = shared.queries;
  RowState<HDP> state[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int32_t r = tile.base + 16 * n + x;
    const bool mine = r < in_seq;
    const int32_t i = mine ? r / group : 0, h = mine ? r - i * group : 0;
    if (wave == n)
      queries.template fill<EXACT>(a, n, static_cast<const uint16_t*>(c.query) + (tile.first + i) * c.query_row_stride +
                                             (head * group + h) * c.query_head_stride, mine);
    state[n].m = -__builtin_inff();
    state[n].l = 0.0f;
#pragma unroll
    for (int l = 0; l < HDP / 16; ++l) state[n].acc[l] = f32x4{0, 0, 0, 0};
  }
  __syncthreads();

  if (token < last) {
    for (;;) {
      const int32_t next = token + kStep;
      f32x4 score[NT][4] = {};
      key_products<0, kDims, HDP, NT, CODEC, DT>(mma, k, queries, score);
      if constexpr (HDP > kDims) {
        load_keys<kDims, EXACT>(a, head_off, token, ids, kDims, k);
        key_products<kDims / 32, kDims, HDP, NT, CODEC, DT>(mma, k, queries, score);
      }
      // Loads return in order: table entries are read two tiles ahead, in front of the keys whose arrival they
      // would else be waited for with.
      GroupIds next_ids;
      GroupEntries later_entries;
      GroupScales next_scales;
      if (next < last) {
        next_ids = group_ids(a, next_entries);
        later_entries = load_entries(a, row, next + kStep, last);
        next_scales = load_scales(c, head, next_ids);
        load_keys<kDims, EXACT>(a, head_off, next, next_ids, 0, k);
      }
      const bool masked = token < all_lo || token + kWaveTokens > all_hi || ballot(!scales.seen) != 0;
      u32x4 p[NT][2][kWeightParts<CODEC, DT>];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        soften<HDP, CODEC>(score[n], queries.factor[n][x], scales, masked, token,
                           [&] { return row_sight(a, tile, before, 16 * n + (lane_now() & 15)); }, state[n]);
        pack_weights<CODEC, DT>(score[n], 0, p[n][0]);
        pack_weights<CODEC, DT>(score[n], 1, p[n][1]);
      }
      value_products<0, kDims, HDP, NT, CODEC, DT>(mma, v, p, state);
      if constexpr (HDP > kDims) {
        load_values<kDims, EXACT>(a, head_off, token, ids, kDims, v);
        value_products<kDims / 16, kDims, HDP, NT, CODEC, DT>(mma, v, p, state);
      }
      if (next >= last) break;
      load_values<kDims, EXACT>(a, head_off, next, next_ids, 0, v);
      ids = next_ids;
      next_entries = later_entries;
      scales = next_scales;
      token = next;
    }
  }

  mma.done();

  const float back = __builtin_ldexpf(1.0f, Mma<CODEC>::kCodeShift - Mma<CODEC>::kWeightTop);
  // The four waves' results of a row are joined by the thread that stores them.
  constexpr int kChunk = HDP < kJoinDims ? HDP : kJoinDims;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float l = groups_sum(state[n].l);
#pragma unroll
    for (int d0 = 0; d0 < HDP; d0 += kChunk) {
      __syncthreads();
      if (lane < 16) {
        shared.ml[wave][x][0] = state[n].m;
        shared.ml[wave][x][1] = l;
      }
#pragma unroll
      for (int k = 0; k < kChunk / 16; ++k)
        *reinterpret_cast<f32x4*>(&shared.joined[wave][x][16 * k + 4 * (lane >> 4)]) = state[n].acc[d0 / 16 + k];
      __syncthreads();
      const int thread = reread(threadIdx.x), at = thread >> 4;
      const int32_t r = tile.base + 16 * n + at;
      if (r >= in_seq) continue;
      const int32_t i = r / group;
      const int64_t rh = static_cast<int64_t>(tile.first + i) * a.heads + head * group + (r - i * group);
      const int64_t part = seg.first_part + (seg.by_row ? rh : 16 * n + at);
      float top = shared.ml[0][at][0];
#pragma unroll
      for (int w = 1; w < kWavesPerBlock; ++w) top = fmaxf(top, shared.ml[w][at][0]);
      const float ref = top == -__builtin_inff() ? 0.0f : top;
      float fade[kWavesPerBlock], sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWavesPerBlock; ++w) {
        fade[w] = __builtin_amdgcn_exp2f(shared.ml[w][at][0] - ref);
        sum += shared.ml[w][at][1] * fade[w];
      }
      for (int k = thread & 15; k < kChunk; k += 16) {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < kWavesPerBlock; ++w) o += shared.joined[w][at][k] * fade[w];
        o *= back;
        if (!EXACT && d0 + k >= a.hd) continue;
        if (seg.parts > 0) {
          if (sum != 0.0f) part_acc(c, seg.parts, part)[d0 + k] = o;
          continue;
        }
        store_o<DT>(c.out, rh * a.hd + d0 + k, sum == 0.0f ? 0.0f : o / sum);
      }
      if (d0 == 0 && (thread & 15) == 0) {
        if (seg.parts > 0) {
          part_ml(c, part)[0] = top;
          part_ml(c, part)[1] = sum;
        } else if (c.lse != nullptr) {
          c.lse[rh] = sum == 0.0f ? -__builtin_inff() : (top + log2f(sum)) * kLn2;
        }
      }
    }
  }
}

// One workgroup per (row tile, kv head, part).
template <int HDP, bool EXACT, int NT, int CODEC, int DT>
__global__ __launch_bounds__(kBlockThreads, rows_occupancy(HDP, EXACT, NT, CODEC))
void attention_rows_kernel(const RowsArgs a) {
  const AttnCall& c = a.c;
  __shared__ RowsShared<HDP, NT, CODEC, DT> shared;
  const int32_t head = blockIdx.y, split = blockIdx.z;
  const RowTile tile = find_tile(a, blockIdx.x, 16 * NT);
  if (c.starts != nullptr && writes_loose_rows(c) && split == 0)
    fill_loose_rows<DT>(c, blockIdx.x, gridDim.x, head * a.group, a.group);
  if (tile.seq < 0) return;
  const Reach reach = tile_reach(a, tile, 16 * NT);
  const Span span = part_span(reach.begin, reach.end, split, a.splits);
  const int64_t per_part = c.rows * c.heads;
  if (a.splits > 1 && span.lo >= span.hi) {  // nothing to do: the rows' parts say so
    const int32_t group = a.group, in_seq = tile.count * group;
    const int32_t r = tile.base + threadIdx.x;
    if (threadIdx.x >= 16 * NT || r >= in_seq) return;
    const int64_t rh = static_cast<int64_t>(tile.first + r / group) * a.heads + head * group + r % group;
    part_ml(c, split * per_part + rh)[0] = -__builtin_inff();
    part_ml(c, split * per_part + rh)[1] = 0.0f;
    return;
  }
  const Segment seg{tile, head, static_cast<int32_t>(span.lo), static_cast<int32_t>(span.hi),
                    a.splits > 1 ? a.splits * per_part : 0, split * per_part, true};
  run_segment<HDP, EXACT, NT, CODEC, DT>(a, seg, reach, shared);
}

// The even cut of a decode step.  Sequences differ in length, so equal parts of each leave most of the chip waiting
// for the longest (64 sequences of 256 to 8192 tokens: 143 us in one part each).
// Here a unit is 256 tokens (a turn of a workgroup's four waves) of a line, one (sequence, row tile, kv head); the lines
// of all sequences stand one behind another, and workgroup i of n takes units [i * all / n, (i + 1) * all / n).
// Only its first line may have begun, and only its last one may go on, in another workgroup: their parts are 2 i
// and 2 i + 1 (times slot_rows); lines in between, or all its own, go to the output at once.
// (Workgroups of one wave, which begin fewer lines each, were no faster at 512 and 2048 lines and slower at 16.)
struct FlowCut {
  uint32_t all, n;
  __device__ __forceinline__ uint32_t start(uint32_t i) const {
    return static_cast<uint32_t>(static_cast<uint64_t>(i) * all / n);
  }
  __device__ __forceinline__ uint32_t owner(uint32_t unit) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(unit + 1) * n - 1) / all);
  }
};

constexpr int32_t kUnitTokens = kWavesPerBlock * kWaveTokens;

__device__ __forceinline__ int32_t reach_turns(const Reach& r) {  // at least one: the row's zeros
  const int32_t n = r.end - r.begin / kWaveTokens * kWaveTokens;
  return r.end > r.begin ? (n + kUnitTokens - 1) / kUnitTokens : 1;
}

__device__ __forceinline__ int32_t seq_turns(const RowsArgs& a, int32_t b) {
  return reach_turns(tile_reach(a, RowTile{b, b, 1, 0}, 1));
}

// A line's sequence, its number within the sequence, the sequence's turns and the line's first unit.  (All units
// together are fewer than 2^31: attention_flows.)
struct FlowLine {
  int32_t seq, line, turns;
  uint32_t first;
};

// Finds the line that holds `unit`; with `all`, the sum of all units is left there instead.
__device__ __forceinline__ FlowLine find_line(const RowsArgs& a, uint32_t lines, uint32_t unit, uint32_t* all) {
  uint32_t before = 0;
  for (int32_t b0 = 0; b0 < a.batch; b0 += kWave) {
    const int32_t b = b0 + lane_id();
    const uint32_t turns = b < a.batch ? seq_turns(a, b) : 0;
    uint32_t end = turns * lines;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint32_t y = __shfl_up(end, o);
      if (lane_id() >= o) end += y;
    }
    end += before;
    const uint64_t hit = ballot(b < a.batch && end > unit);
    if (all == nullptr && hit != 0) {
      const int src = __builtin_ctzll(hit);
      FlowLine found;
      found.seq = b0 + src;
      found.turns = __builtin_amdgcn_readlane(turns, src);
      const uint32_t base = __builtin_amdgcn_readlane(end, src) - found.turns * lines;
      found.line = static_cast<int32_t>((unit - base) / static_cast<uint32_t>(found.turns));
      found.first = base + static_cast<uint32_t>(found.line) * found.turns;
      return found;
    }
    before = __builtin_amdgcn_readlane(end, kWave - 1);
  }
  if (all != nullptr) *all = before;
  return {-1, 0, 1, 0};
}

__device__ __forceinline__ FlowCut flow_cut(uint32_t all, uint32_t groups) { return {all, all < groups ? all : groups}; }

template <int HDP, bool EXACT, int NT, int CODEC, int DT>
__global__ __launch_bounds__(kBlockThreads, rows_occupancy(HDP, EXACT, NT, CODEC))
void attention_flow_kernel(const RowsArgs a) {
  __shared__ RowsShared<HDP, NT, CODEC, DT> shared;
  const uint32_t lines = static_cast<uint32_t>(a.heads / a.group) * a.seq_tiles;
  // This workgroup's units to come and the line that they begin in (in registers they would be held over a segment).
  __shared__ struct {
    uint32_t unit, end, first, all;
    int32_t seq, line;
  } share;
  {
    uint32_t all = 0;
    find_line(a, lines, 0, &all);
    const FlowCut cut = flow_cut(all, gridDim.x);
    if (blockIdx.x >= cut.n) return;
    const uint32_t unit = cut.start(blockIdx.x);
    const FlowLine line = find_line(a, lines, unit, nullptr);
    if (threadIdx.x == 0) share = {unit, cut.start(blockIdx.x + 1), line.first, all, line.seq, line.line};
  }
  for (;;) {
    __syncthreads();
    const uint32_t unit = __builtin_amdgcn_readfirstlane(share.unit), end = __builtin_amdgcn_readfirstlane(share.end);
    const uint32_t first = __builtin_amdgcn_readfirstlane(share.first);
    const int32_t seq = __builtin_amdgcn_readfirstlane(share.seq), line = __builtin_amdgcn_readfirstlane(share.line);
    if (unit >= end) return;
    const int32_t head = line / a.seq_tiles, tile_no = line - head * a.seq_tiles;
    const RowTile tile{seq, seq, 1, tile_no * 16 * NT};
    const Reach reach = tile_reach(a, tile, 16 * NT);
    const int32_t turns = reach_turns(reach), turn = static_cast<int32_t>(unit - first);
    const int32_t take = min(static_cast<int32_t>(end - unit), turns - turn);
    const int32_t lo = reach.begin / kWaveTokens * kWaveTokens + turn * kUnitTokens;
    const bool whole = take == turns;
    const Segment seg{tile, head, lo, min(reach.end, lo + take * kUnitTokens),
                      whole ? 0 : int64_t{2} * gridDim.x * a.slot_rows,
                      (int64_t{2} * blockIdx.x + (turn == 0)) * a.slot_rows, false};
    __syncthreads();  // every wave has read its share
    if (threadIdx.x == 0) {
      const bool same = line + 1 < static_cast<int32_t>(lines);
      share.unit = unit + take;
      share.first = first + turns;
      share.seq = same ? seq : seq + 1;
      share.line = same ? line + 1 : 0;
      if (turn == 0) {
        uint32_t* owners = line_owners(a.c, int64_t{2} * gridDim.x * a.slot_rows, static_cast<int64_t>(seq) * lines + line);
        owners[0] = blockIdx.x;
        owners[1] = whole ? blockIdx.x : flow_cut(share.all, gridDim.x).owner(first + turns - 1);
      }
    }
    run_segment<HDP, EXACT, NT, CODEC, DT>(a, seg, reach, shared);
  }
}

// ----- joining the parts: one workgroup per (row, head) ---------------------------------------------
// Lane j holds the maximum and sum of part j of a round of 64; the waves add up the parts' results by turns, and the
// first one stores their sum.  Parts that saw nothing hold no result: what is read in its place is not used.
constexpr int kMostSplits = 64;

// The parts of a (row, head): part j is first + j * step, but part 0 of an even cut is its own.
struct PartList {
  int64_t count, total, zeroth, first, step;
  __device__ __forceinline__ int64_t at(int64_t j) const { return j == 0 ? zeroth : first + j * step; }
};

// WAVES of the workgroup add up one (row, head) together.
template <int DT, int WAVES>
__device__ __forceinline__ void join_parts(const AttnCall& c, int64_t rh, const PartList& parts) {
  const int lane = lane_id(), wave = WAVES > 1 ? wave_in_block() : 0;
  const int hd = static_cast<int>(c.head_dim);
  float top = -__builtin_inff();
  for (int64_t j = lane; j < parts.count; j += kWave) top = fmaxf(top, part_ml(c, parts.at(j))[0]);
  top = wave_max(top);
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  float sum = 0.0f;
  float acc[kAnyMaxDim / kWave] = {};
  for (int64_t j0 = 0; j0 < parts.count; j0 += kWave) {
    float m = -__builtin_inff(), l = 0.0f;
    if (j0 + lane < parts.count) {
      m = part_ml(c, parts.at(j0 + lane))[0];
      l = part_ml(c, parts.at(j0 + lane))[1];
    }
    const float fade = __builtin_amdgcn_exp2f(m - ref);
    sum += wave_sum(l * fade);
    const int64_t left = parts.count - j0;
    const int round = left < kWave ? static_cast<int>(left) : kWave;
    for (int s0 = wave; s0 < round; s0 += 4 * WAVES) {
      float f[4], part[4][kAnyMaxDim / kWave];
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // four parts on their way at a time
        const int s = s0 + u * WAVES < round ? s0 + u * WAVES : s0;
        const bool used = s0 + u * WAVES < round &&
                          __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(l), s)) != 0.0f;
        f[u] = used ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(fade), s)) : 0.0f;
        const float* p = part_acc(c, parts.total, parts.at(j0 + s));
#pragma unroll
        for (int i = 0; i < kAnyMaxDim / kWave; ++i) {
          part[u][i] = 0.0f;
          if (i * kWave < hd && lane + i * kWave < hd) part[u][i] = p[lane + i * kWave];
          if (!used) part[u][i] = 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < kAnyMaxDim / kWave; ++i) acc[i] = __builtin_fmaf(part[u][i], f[u], acc[i]);
    }
  }
  if constexpr (WAVES > 1) {
    __shared__ float sums[WAVES - 1][kAnyMaxDim];
    if (wave > 0)
#pragma unroll
      for (int i = 0; i < kAnyMaxDim / kWave; ++i)
        if (lane + i * kWave < hd) sums[wave - 1][lane + i * kWave] = acc[i];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int i = 0; i < kAnyMaxDim / kWave; ++i)
      if (lane + i * kWave < hd)
        for (int w = 0; w < WAVES - 1; ++w) acc[i] += sums[w][lane + i * kWave];
  }
#pragma unroll
  for (int i = 0; i < kAnyMaxDim / kWave; ++i)
    if (lane + i * kWave < hd) store_o<DT>(c.out, rh * hd + lane + i * kWave, sum == 0.0f ? 0.0f : acc[i] / sum);
  if (c.lse != nullptr && lane == 0) c.lse[rh] = sum == 0.0f ? -__builtin_inff() : (top + log2f(sum)) * kLn2;
}

// A workgroup per (row, head), or with WAVES 1 a wave (many rows, few parts of each).
constexpr int64_t kWaveJoinRows = 512;

template <int DT, int WAVES>
__global__ __launch_bounds__(kBlockThreads) void attention_join_kernel(const AttnCall c) {
  const int64_t rh = WAVES > 1 ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave_in_block();
  const int64_t per_part = c.rows * c.heads;
  if (rh >= per_part || row_sequence(c, rh / c.heads).seq < 0) return;  // no parts
  join_parts<DT, WAVES>(c, rh, {c.splits, c.splits * per_part, rh, rh, per_part});
}

// Lines that lie in one workgroup's share are done.
template <int DT, int WAVES>
__global__ __launch_bounds__(kBlockThreads) void attention_flow_join_kernel(const RowsArgs a, uint32_t groups,
                                                                           int32_t tile_rows) {
  const uint32_t rh = WAVES > 1 ? blockIdx.x : blockIdx.x * kWavesPerBlock + wave_in_block();
  if (rh >= static_cast<uint32_t>(a.batch) * a.heads) return;
  const int32_t seq = rh / a.heads, hq = rh - seq * a.heads;
  const int32_t head = hq / a.group, r = hq - head * a.group, tile = r / tile_rows;
  const int64_t rows = a.slot_rows, total = 2 * groups * rows, in_tile = r - tile * tile_rows;
  const int64_t line = (static_cast<int64_t>(seq) * (a.heads / a.group) + head) * a.seq_tiles + tile;
  const uint32_t* owners = line_owners(a.c, total, line);
  const int64_t from = __builtin_amdgcn_readfirstlane(owners[0]), to = __builtin_amdgcn_readfirstlane(owners[1]);
  if (from == to) return;
  join_parts<DT, WAVES>(a.c, rh, {to - from + 1, total, (2 * from + 1) * rows + in_tile, 2 * from * rows + in_tile, 2 * rows});
}

template <int DT>
hipError_t launch_join(const AttnCall& c, hipStream_t stream) {
  const int64_t rh = c.rows * c.heads;
  if (rh < kWaveJoinRows)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_join_kernel<DT, kWavesPerBlock>), dim3(static_cast<uint32_t>(rh)),
                       dim3(kBlockThreads), 0, stream, c);
  else
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_join_kernel<DT, 1>),
                       dim3(static_cast<uint32_t>((rh + kWavesPerBlock - 1) / kWavesPerBlock)), dim3(kBlockThreads), 0,
                       stream, c);
  return hipGetLastError();
}

template <int DT, int CODEC>
hipError_t launch_any(const AttnCall& c, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(c.rows), static_cast<uint32_t>(c.heads), static_cast<uint32_t>(c.splits));
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_any_kernel<DT, CODEC>), grid, dim3(kBlockThreads), 0, stream, c);
  return hipGetLastError();
}

// Whether the matrix-core form takes the call: 16-bit queries, up to 256 dims, 16-token groups that lie in one
// block and begin at multiples of 16 bytes, places in a block and head that 32 bits hold.
bool takes_rows(const AttnCall& c) {
  if (c.dtype == kLinF32 || c.head_dim > 256 || c.block_size % 16 != 0 || c.head_dim * c.block_size >= 1 << 30)
    return false;
  uint64_t all = 0;
  for (int kv = 0; kv < 2; ++kv)
    all |= reinterpret_cast<uint64_t>(c.cache[kv]) | static_cast<uint64_t>(c.cache_block_stride[kv]);
  return all % 16 == 0;
}

// 16-row tiles that a wave holds: 2 where the rows of a sequence fill more than one on average and two fit the
// registers.
int row_tiles(const AttnCall& c) {
  if (c.head_dim > 128) return 1;
  const int64_t group = c.heads / c.kv_heads;
  const int64_t rows = c.starts == nullptr ? 1 : c.batch > 0 ? (c.rows + c.batch - 1) / c.batch : 1;
  return rows * group <= 16 ? 1 : 2;
}

constexpr int64_t kComputeUnits = 256;

// Whether prompt chunks' form (kv_attention_wide.hip) takes the call.  It decodes a token tile once for 128 rows, the
// other form for every 16 or 32, but goes through the tokens of a part one tile at a time where the other one's waves
// take four at once.  Rows are those of a kv head and sequence, on average: 32 x 96 rows against 2000 tokens 80 us, the
// other form 118, 8 x 128 against 4096 tokens 60 against 70, 8 x 68: 48 against 67; 32 x 36 rows 73 against 77, but with 64
// dims (64 x 40 rows) 84 against 65.
bool takes_wide(const AttnCall& c) {
  return takes_rows(c) && c.starts != nullptr && c.head_dim <= 128 && c.batch > 0 &&
         (c.rows + c.batch - 1) / c.batch * (c.heads / c.kv_heads) > 64;
}

// How an even cut is made: workgroups (what the chip holds at once, or one for each unit that the tables have room
// for) and rows of a part.
struct FlowPlan {
  int64_t groups, slot_rows;
};

// Workgroups of the rows and flow kernels that a CU holds.
int held_by_a_unit(const AttnCall& c) {
  const int hdp = c.head_dim <= 64 ? 64 : c.head_dim == 96 ? 96 : c.head_dim <= 128 ? 128 : 256;
  return rows_occupancy(hdp, c.head_dim == hdp, row_tiles(c), c.codec);
}

FlowPlan flow_plan(const AttnCall& c) {
  const int tiles = row_tiles(c), size = 16 * tiles;
  const int64_t lines = tiles_bound(c, size) * c.kv_heads, group = c.heads / c.kv_heads;
  const int64_t turns = (c.max_blocks * c.block_size + kUnitTokens - 1) / kUnitTokens;
  const int64_t most = lines * (turns > 0 ? turns : 1);
  const int64_t held = kComputeUnits * held_by_a_unit(c);
  return {most < held ? most : held, group < size ? group : size};
}

template <int HDP, bool EXACT, int NT, int CODEC, int DT>
hipError_t launch_rows_as(const AttnCall& c, hipStream_t stream) {
  RowsArgs a = rows_args(c, 16 * NT);
  if (c.splits == 0) {
    const FlowPlan plan = flow_plan(c);
    const uint32_t groups = static_cast<uint32_t>(plan.groups);
    a.slot_rows = static_cast<int32_t>(plan.slot_rows);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_flow_kernel<HDP, EXACT, NT, CODEC, DT>), dim3(groups),
                       dim3(kBlockThreads), 0, stream, a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    const int64_t rh = c.rows * c.heads;
    if (rh < kWaveJoinRows)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_flow_join_kernel<DT, kWavesPerBlock>),
                         dim3(static_cast<uint32_t>(rh)), dim3(kBlockThreads), 0, stream, a, groups, 16 * NT);
    else
      hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_flow_join_kernel<DT, 1>),
                         dim3(static_cast<uint32_t>((rh + kWavesPerBlock - 1) / kWavesPerBlock)), dim3(kBlockThreads),
                         0, stream, a, groups, 16 * NT);
    return hipGetLastError();
  }
  int64_t tiles = tiles_bound(c, 16 * NT);
  if (tiles < 1) tiles = 1;  // rows of no sequence are still to be filled
  const dim3 grid(static_cast<uint32_t>(tiles), static_cast<uint32_t>(c.kv_heads), static_cast<uint32_t>(c.splits));
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_rows_kernel<HDP, EXACT, NT, CODEC, DT>), grid, dim3(kBlockThreads), 0,
                     stream, a);
  return hipGetLastError();
}

template <int DT, int CODEC, int NT>
hipError_t launch_rows(const AttnCall& c, hipStream_t stream) {
  if (c.head_dim == 64) return launch_rows_as<64, true, NT, CODEC, DT>(c, stream);
  if (c.head_dim < 64) return launch_rows_as<64, false, NT, CODEC, DT>(c, stream);
  if (c.head_dim == 96) return launch_rows_as<96, true, NT, CODEC, DT>(c, stream);
  if (c.head_dim == 128) return launch_rows_as<128, true, NT, CODEC, DT>(c, stream);
  if (c.head_dim < 128) return launch_rows_as<128, false, NT, CODEC, DT>(c, stream);
  if (c.head_dim == 256) return launch_rows_as<256, true, 1, CODEC, DT>(c, stream);
  return launch_rows_as<256, false, 1, CODEC, DT>(c, stream);
}

template <int DT, int CODEC>
hipError_t launch_typed(const AttnCall& c, hipStream_t stream) {
  if constexpr (DT != kLinF32) {
    if (takes_wide(c)) return launch_wide(c, stream);
    if (takes_rows(c))
      return row_tiles(c) == 1 ? launch_rows<DT, CODEC, 1>(c, stream) : launch_rows<DT, CODEC, 2>(c, stream);
  }
  return launch_any<DT, CODEC>(c, stream);
}

template <int DT>
hipError_t launch_dtype(const AttnCall& c, hipStream_t stream) {
  const hipError_t err = c.codec == kE4M3 ? launch_typed<DT, kE4M3>(c, stream) : launch_typed<DT, kE5M2>(c, stream);
  if (err != hipSuccess || c.splits <= 1) return err;
  return launch_join<DT>(c, stream);
}

}  // namespace

bool attention_flows(const AttnCall& c) {
  const int64_t turns = c.max_blocks * c.block_size / kWaveTokens + 2;
  return c.starts == nullptr && c.batch > 0 && takes_rows(c) &&
         c.batch < (int64_t{1} << 31) / turns / (c.kv_heads + c.heads);
}

// How a call is cut.  Decode steps of sequences longer than kFlowFrom: evenly (0).  An even cut costs its join and its
// search and gains where lengths differ: 64 rows of 64 to 8192 tokens 117 us, by parts 134; of 64 to 4000 62 against 64;
// of 64 to 2000 43 against 38; and where all are equally long, 4096, 116 against 103.
// Others: as many parts as give the chip's CUs two workgroups each, or one where a CU holds no more, in whole turns of
// 256 tokens (8 rows of 1000 tokens: 12.9 us in four parts, 16.1 in one; 64 rows: 26.5 in one, 33 in two; 32 x 32
// rows, one workgroup a CU: 42 in one, 58 in two).  Up to 512 tokens: one (8 rows of 500: 11.0 us, in two parts 12.6);
// prompt chunks, whose many rows make parts dear, up to 1024 (1000 rows of 4 heads against 1000 tokens: 40 us, in two
// parts 54; 64 rows against 2000: 66, in eight 24).
constexpr int64_t kFlowFrom = 4096;

// Tokens of a sequence of at most `longest` that a row tile goes through: with a window, its rows' windows side by side
// from the tile of tokens on in which the first one begins.  (64 decode rows of 256 to 8192 tokens with a window of 1000:
// 30.6 us, cut by their lengths 42.9; 8 x 8 draft rows far behind a window of 256: 13.4, by lengths 18.0.)
int64_t tile_span_bound(const AttnCall& c, int64_t longest) {
  if (c.window <= 0 || c.window >= longest) return longest;
  const int64_t rows = takes_wide(c) ? kWideRows : takes_rows(c) ? 16 * row_tiles(c) : 1;
  const int64_t group = c.heads / c.kv_heads, positions = c.starts == nullptr ? 1 : (rows + group - 2) / group + 1;
  const int64_t span = c.window + positions + kPartTokens - 2;
  return span < longest ? span : longest;
}

int64_t attention_splits(const AttnCall& c, int64_t longest) {
  longest = tile_span_bound(c, longest);
  if (attention_flows(c) && longest > kFlowFrom) return 0;
  int64_t groups = c.rows * c.heads, wanted = 4 * kComputeUnits;
  if (takes_wide(c)) {
    groups = tiles_bound(c, kWideRows) * c.kv_heads;
    wanted = 2 * kComputeUnits;
  } else if (takes_rows(c)) {
    groups = tiles_bound(c, 16 * row_tiles(c)) * c.kv_heads;
    wanted = kComputeUnits * (held_by_a_unit(c) > 1 ? 2 : 1);
  }
  const int64_t whole = takes_wide(c) ? 4 * kTurnTokens : 2 * kTurnTokens;
  const int64_t most = longest <= whole ? 1 : (longest - 1) / kTurnTokens + 1;
  int64_t splits = groups > 0 ? wanted / groups : 1;
  splits = splits < most ? splits : most;
  splits = splits < 1 ? 1 : splits > kMostSplits ? kMostSplits : splits;
  const int64_t per = (most + splits - 1) / splits;
  return (most + per - 1) / per;  // none that would be left without a turn
}

int64_t attention_workspace(const AttnCall& c) {
  if (c.splits == 1) return 0;
  int64_t parts = c.splits * c.rows * c.heads;
  if (c.splits == 0) {
    const FlowPlan plan = flow_plan(c);
    parts = 2 * plan.groups * plan.slot_rows;
    return 4 * parts * (c.head_dim + 2) + 8 * tiles_bound(c, 16 * row_tiles(c)) * c.kv_heads;
  }
  return 4 * parts * (c.head_dim + 2);
}

hipError_t launch_attention(const AttnCall& c, hipStream_t stream) {
  switch (c.dtype) {
    case kLinF32: return launch_dtype<kLinF32>(c, stream);
    case kLinF16: return launch_dtype<kLinF16>(c, stream);
    case kLinBF16: return launch_dtype<kLinBF16>(c, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace kvhip
