// Attention over a paged FP8 cache with block scales (see kv_attention.hip) for many query rows: prompt chunks.
//
// There the matrix products and what stands between them bound the work, not the cache: a 64-token tile of 128 dims
// costs a wave of 32 rows 1024 cycles of matrix instructions, and turning its codes into 16-bit floats 1900.  So a
// workgroup's four waves take 32 rows each of one row tile, decode a quarter of every token tile each, and leave it
// in LDS in the order in which matrix instructions read it, for all four; two such buffers, and one barrier a tile.
//
// S^T = K Q^T and O^T += V^T P^T with 32x32x16 instructions, whose results give lane (x = lane % 32, h = lane / 32)
// of column x the rows 8 (r / 4) + 4 h + r % 4, r = 0..15.  Row 8 a + 4 h + b of K's operand is token 16 h + 4 a + b
// of its 32, so the lane holds tokens 16 h + r of query row x: one 16-token group, which lies in one block (scales
// and masks are per lane), in the order in which V's operand, 8 tokens a lane, wants the weights.  Nothing crosses
// lanes but the running maximum.  The rest (codes, scaling of queries and weights) is as in kv_attention.hip.
//
// Chunks of 2048 and 1753 rows (32 heads, 8 kv heads, 128 dims; 3769 and 8192 cached tokens): 413 to 430 us, 750 to 785
// TFLOP/s; 8192 rows against 16384 tokens: 1920 to 1980 us, 830 to 860 TFLOP/s (a large library product of bf16 matrices: 1260).  The first dozen calls
// after a pause take 530 us.  The instructions of a wave's tile (1024 cycles of matrix instructions, about 1900 of others, a
// third of them exponentials) bound it; the two waves of a SIMD mostly take turns: 31% and 57% of its cycles.  Tried and
// slower or no faster: 256-row tiles of eight waves (6% faster for the largest calls, 5 to 25% slower elsewhere), the next
// tile's score products among this tile's exponentials (their registers leave one wave per SIMD: 800 us), wave priorities.
#include "kv_attention.h"

namespace kvhip {
namespace attn {
namespace {

using f32x16 = float __attribute__((ext_vector_type(16)));

constexpr int kTileTokens = 64;
// The maximum that weights are taken relative to stays behind the running one by up to a factor of two, which their
// 16 bits have place for: the sums so far are rescaled less often.
constexpr float kLag = 1.0f;
// A product with the scales that is not rounded may pass a maximum that is, by half a step of it.  Past kFusedScores
// products are rounded first, and the maximum stays behind by nothing: m + 1 is no number among steps of 2.
constexpr float kFusedScores = 0x1p22f;
constexpr int kWaveRows = 32;
static_assert(kWideRows == kWaveRows * kWavesPerBlock && kTileTokens == 16 * kWavesPerBlock, "a wave decodes one group");


template <int CODEC>
__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (CODEC == kE4M3)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The sum or maximum of both half waves' values.
__device__ __forceinline__ float other_half(float v) {
  const uint32_t b = __float_as_uint(v);
  const auto s = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return __uint_as_float(lane_id() < 32 ? s[1] : s[0]);
}

// A token tile's operands.  k: [32 tokens][16 dims][slot], the slots of a 1-KB operand permuted so that neither the
// lanes that write tokens 4 apart nor those that read neighbours meet in a bank.  v: [32 tokens][16 of them in
// halves][32 dims][lane].  Scales of the four groups: key, value, and 1 if the group has a block.
template <int HDP>
struct TokenTile {
  u32x4 k[2][HDP / 16][kWave];
  u32x4 v[2][2][HDP / 32][kWave];
  f32x4 scales[4];
};

// Slot of row 8 a + 4 h0 + b, dims half h.
__device__ __forceinline__ int key_slot(int a, int h0, int b, int h) {
  return 32 * h + 8 * a + (((4 * h0) | (b ^ a)) ^ (4 * h));
}

// A wave's group of 16 tokens: codes on their way from the cache.  Octet o of the dims is d = o + j * HDP / 8.
template <int HDP>
struct GroupCodes {
  uint32_t k[8];          // tokens 4 (lane % 4) .. + 3 of octet lane / 4
  u32x4 v[HDP / kWave];   // 16 tokens of dim lane + 64 e
  float ks, vs;
  bool seen;
};

template <int HDP, bool EXACT>
__device__ __forceinline__ void load_group(const RowsArgs& a, int32_t head, int32_t token, int32_t block,
                                           GroupCodes<HDP>& codes) {
  const AttnCall& c = a.c;
  const int lane = lane_id();
  // Addresses are a scalar (the block is the same for the wave) and 32 bits of a lane.  A group without a block reads
  // block 0, which every cache has; its scores are masked.
  const int64_t blk = block < 0 ? 0 : block;
  const int64_t off = static_cast<int64_t>(head) * a.hd * a.bs + group_place(a, token);
  const uint8_t* k = static_cast<const uint8_t*>(c.cache[0]) + blk * c.cache_block_stride[0] + off;
  const uint8_t* v = static_cast<const uint8_t*>(c.cache[1]) + blk * c.cache_block_stride[1] + off;
  const int octet = (lane >> 2) & (HDP / 8 - 1), quad = lane & 3, last = a.hd - 1;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t at = (EXACT ? octet : min(octet + j * (HDP / 8), last)) * a.bs + 4 * quad;
    codes.k[j] = load4(k + (EXACT ? j * (HDP / 8) * a.bs : 0) + at);
  }
#pragma unroll
  for (int e = 0; e < HDP / kWave; ++e) {
    const uint32_t at = (EXACT ? lane : min(lane + e * kWave, last)) * a.bs;
    codes.v[e] = ld16_cached(v + (EXACT ? e * kWave * a.bs : 0) + at);
  }
  codes.ks = c.scale[0][blk * c.scale_block_stride[0] + head * c.scale_head_stride[0]];
  codes.vs = c.scale[1][blk * c.scale_block_stride[1] + head * c.scale_head_stride[1]];
  codes.seen = block >= 0;
}

template <int HDP, int CODEC>
__device__ __forceinline__ void decode_group(const Mma<CODEC>& mma, const GroupCodes<HDP>& codes, TokenTile<HDP>& tile) {
  const int lane = lane_now(), wave = wave_in_block(), p = wave >> 1, h0 = wave & 1;
  const int octet = lane >> 2, quad = lane & 3;
  if (HDP / 8 * 4 == kWave || octet < HDP / 8) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = mma.prepare(codes.k[j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 o;
      // Bytes i of rows j and j + 1 into the high bytes of the halves.
      const uint32_t sel = 0x000C000Cu | (static_cast<uint32_t>(i) << 8) | (static_cast<uint32_t>(4 + i) << 24);
#pragma unroll
      for (int j = 0; j < 8; j += 2) o[j / 2] = mma.pair(__builtin_amdgcn_perm(w[j + 1], w[j], sel));
      tile.k[p][octet >> 1][key_slot(quad, h0, i, octet & 1)] = o;
    }
  }
#pragma unroll
  for (int e = 0; e < HDP / kWave; ++e) {
    const int d = lane + e * kWave;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      u32x4 o;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t w = mma.prepare(codes.v[e][2 * half + x]);
        o[2 * x] = mma.pair(w << 8);
        o[2 * x + 1] = mma.pair(w);
      }
      tile.v[p][half][d >> 5][(d & 31) + 32 * h0] = o;
    }
  }
  if (lane == 0) tile.scales[wave] = f32x4{codes.ks, codes.vs, codes.seen ? 1.0f : 0.0f, 0.0f};
}

// A lane's query row, in registers: element j of step s is d = 2 s + h + j * HDP / 8.  Returns the factor of its
// scores.
template <int HDP, bool EXACT, int CODEC, int DT>
__device__ __forceinline__ float read_query(const RowsArgs& a, const uint16_t* row, bool mine,
                                            u32x4 (*q)[HDP / 16]) {
  const int h = lane_id() >> 5;
  uint16_t raw[HDP / 16][8];
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (EXACT) {
#pragma unroll
      for (int e = 0; e < HDP / 64; ++e) {
        const u32x4 piece = *reinterpret_cast<const u32x4*>(row + j * (HDP / 8) + 8 * e);
#pragma unroll
        for (int s = 0; s < 4; ++s)
          raw[4 * e + s][j] = mine ? static_cast<uint16_t>(h != 0 ? piece[s] >> 16 : piece[s]) : 0;
      }
    } else {
#pragma unroll
      for (int s = 0; s < HDP / 16; ++s) {
        const int d = 2 * s + h + j * (HDP / 8);
        raw[s][j] = row[min(d, a.hd - 1)];
        if (!mine || d >= a.hd) raw[s][j] = 0;
      }
    }
#pragma unroll
    for (int s = 0; s < HDP / 16; ++s) most = fmaxf(most, fabsf(query_value<DT>(raw[s][j])));
  }
  most = fmaxf(most, other_half(most));
  const bool fine = most > 0.0f && most < __builtin_inff();
  const int up = fine ? Mma<CODEC>::kQueryTop - ilogbf(most) : 0;
#pragma unroll
  for (int s = 0; s < HDP / 16; ++s)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float lo = __builtin_ldexpf(query_value<DT>(raw[s][j]), up), hi = __builtin_ldexpf(query_value<DT>(raw[s][j + 1]), up);
#pragma unroll
      for (int part = 0; part < kQueryParts<CODEC, DT>; ++part) {
        q[part][s][j / 2] = Mma<CODEC>::pack(lo, hi);
        const f32x2 took = Mma<CODEC>::unpack(q[part][s][j / 2]);
        lo -= took[0];
        hi -= took[1];
      }
    }
  return __builtin_ldexpf(static_cast<float>(a.c.softmax_scale) * kLog2e, Mma<CODEC>::kCodeShift - up);
}


template <int HDP, bool EXACT, int CODEC, int DT>
__global__ __launch_bounds__(kBlockThreads, 2)
void attention_wide_kernel(const RowsArgs a, uint32_t tiles) {
  const AttnCall& c = a.c;
  __shared__ TokenTile<HDP> buffer[2];
  // Workgroups go over the chip by turns: neighbours are heads of one row tile, and the tiles that see most of a
  // sequence come first.
  const uint32_t kv_heads = static_cast<uint32_t>(a.heads / a.group);
  const uint32_t at = blockIdx.x / kv_heads;
  const int32_t head = static_cast<int32_t>(blockIdx.x - at * kv_heads), split = static_cast<int32_t>(at % a.splits);
  const int32_t index = static_cast<int32_t>(tiles - 1 - at / a.splits);
  const int32_t group = a.group;
  const RowTile tile = find_tile(a, index, kWideRows);
  if (c.starts != nullptr && writes_loose_rows(c) && split == 0)
    fill_loose_rows<DT>(c, index, tiles, head * group, group);
  if (tile.seq < 0) return;
  const Reach reach = tile_reach(a, tile, kWideRows);
  const Span span = part_span(reach.begin, reach.end, split, a.splits);
  const int32_t in_seq = tile.count * group;
  const int lane = lane_id(), x = lane & 31, h = lane >> 5, wave = wave_in_block();
  const uint8_t* table = static_cast<const uint8_t*>(c.tables) + tile.seq * c.table_stride * (c.wide_tables ? 8 : 4);

  const int32_t last = static_cast<int32_t>(span.hi);
  // Tiles of tokens inside [all_lo, all_hi) are seen whole by every row.
  const int32_t all_lo = a.window > 0 ? max(reach.pos_hi - a.window + 1, 0) : 0;
  const int32_t all_hi = min(reach.pos_lo + 1, last);
  int32_t token = static_cast<int32_t>(span.lo);
  const int mine_at = 16 * wave;  // the wave's group in a tile
  GroupCodes<HDP> codes;
  Entry next_entry;
  if (token < last) {
    const Entry entry = load_first_entry(a, table, token + mine_at, reach.begin, last);
    next_entry = load_entry(a, table, token + kTileTokens + mine_at, last);
    load_group<HDP, EXACT>(a, head, token + mine_at, __builtin_amdgcn_readfirstlane(entry_block(a, entry)), codes);
  }

  const Mma<CODEC> mma;
  constexpr int kParts = kWeightParts<CODEC, DT>;
  const int32_t r0 = tile.base + kWaveRows * wave + x;
  const bool mine = r0 < in_seq;
  const int32_t row_i = mine ? r0 / group : 0, row_h = mine ? r0 - row_i * group : 0;
  const int32_t pos = reach.before + row_i;
  u32x4 q[kQueryParts<CODEC, DT>][HDP / 16];
  const float factor = read_query<HDP, EXACT, CODEC, DT>(
      a, static_cast<const uint16_t*>(c.query) + (tile.first + row_i) * c.query_row_stride +
             (head * group + row_h) * c.query_head_stride, mine, q);
  const int32_t sight_hi = mine ? min(pos + 1, a.room) : 0;
  const int32_t sight_lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;

  f32x16 acc[HDP / 32] = {};
  float m = -__builtin_inff(), l = 0.0f;
  bool coarse = false;  // some row's m
  if (token < last) {
    decode_group<HDP, CODEC>(mma, codes, buffer[0]);
    if (token + kTileTokens < last) {
      const int32_t block = __builtin_amdgcn_readfirstlane(entry_block(a, next_entry));
      next_entry = load_entry(a, table, token + 2 * kTileTokens + mine_at, last);
      load_group<HDP, EXACT>(a, head, token + kTileTokens + mine_at, block, codes);
    }
  }
  __syncthreads();
  int now = 0;
  const int read_slot = key_slot(x >> 3, (x >> 2) & 1, x & 3, h);
  for (; token < last; token += kTileTokens, now ^= 1) {
    const TokenTile<HDP>& t = buffer[now];
    f32x16 score[2] = {};
#pragma unroll
    for (int s = 0; s < HDP / 16; ++s)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const u32x4 k = t.k[p][s][read_slot];
#pragma unroll
        for (int part = 0; part < kQueryParts<CODEC, DT>; ++part) score[p] = mma32<CODEC>(k, q[part][s], score[p]);
      }
    // Operands on their way three products ahead.
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
    for (int i = 0; i < HDP / 16 - 3; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 6, 0);
    // The next tile, into the buffer that was read before the last barrier.
    if (token + kTileTokens < last) {
      decode_group<HDP, CODEC>(mma, codes, buffer[now ^ 1]);
      if (token + 2 * kTileTokens < last) {
        const int32_t block = __builtin_amdgcn_readfirstlane(entry_block(a, next_entry));
        next_entry = load_entry(a, table, token + 3 * kTileTokens + mine_at, last);
        load_group<HDP, EXACT>(a, head, token + 2 * kTileTokens + mine_at, block, codes);
      }
    }

    const f32x4 scales[2] = {t.scales[h], t.scales[2 + h]};
    float f[2] = {factor * scales[0][0], factor * scales[1][0]};
    // The maximum of the scores is the factor times that of the products where no factor is negative.
    if (token < all_lo || token + kTileTokens > all_hi || factor < 0.0f ||
        ballot(scales[0][2] * scales[1][2] == 0.0f) != 0) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int first = token + 32 * p + 16 * h;
        const int lo = sight_lo - first, hi = scales[p][2] != 0.0f ? sight_hi - first : 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) score[p][r] = r < lo || r >= hi ? -__builtin_inff() : score[p][r] * f[p];
        f[p] = 1.0f;
      }
    }
    float most[2], lift[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      most[p] = score[p][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) most[p] = fmaxf(most[p], score[p][r]);
      lift[p] = score_lift(0.0f, scales[p][1]);
    }
    // For a maximum that is coarse: past kFusedScores.
    auto round_products = [&] {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        score[p] *= f[p];
        most[p] *= f[p];
        lift[p] = score_lift(most[p], scales[p][1]);
        f[p] = 1.0f;
      }
    };
    auto highest = [&] {
      const float top = fmaxf(m, fmaxf(__builtin_fmaf(most[0], f[0], lift[0]), __builtin_fmaf(most[1], f[1], lift[1])));
      return fmaxf(top, other_half(top));
    };
    if (coarse) round_products();
    float top = highest();
    if (ballot(top > m + (coarse ? 0.0f : kLag)) != 0) {
      // A maximum becomes coarse only here.  (Looked for in every tile it took 2% more time.)
      if (!coarse && ballot(fabsf(top) > kFusedScores && top > -__builtin_inff()) != 0) {
        coarse = true;
        round_products();
        top = highest();
      }
      const float fade = __builtin_amdgcn_exp2f(m - (top == -__builtin_inff() ? 0.0f : top));
      l *= fade;
#pragma unroll
      for (int i = 0; i < HDP / 32; ++i) acc[i] *= fade;
      m = top;
    }
    const float ref = m == -__builtin_inff() ? 0.0f : m;
    u32x4 w[2][2][kParts];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const float weight = scales[p][2] != 0.0f ? __builtin_ldexpf(scales[p][1], Mma<CODEC>::kWeightTop) : 0.0f;
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(score[p][r], f[p], -ref));
        sum += e;
        score[p][r] = e * weight;
      }
      l += sum;
      // Tokens (0, 2), (1, 3) of a dword, as codes come out of theirs.
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * half + 4 * (i >> 1) + (i & 1);
          float lo = score[p][r], hi = score[p][r + 2];
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            w[p][half][part][i] = Mma<CODEC>::pack(lo, hi);
            const f32x2 took = Mma<CODEC>::unpack(w[p][half][part][i]);
            lo -= took[0];
            hi -= took[1];
          }
        }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < HDP / 32; ++i) {
          const u32x4 v = t.v[p][half][i][lane];
#pragma unroll
          for (int part = 0; part < kParts; ++part) acc[i] = mma32<CODEC>(v, w[p][half][part], acc[i]);
        }
    __syncthreads();
  }
  mma.done();

  if (!mine) return;
  const float back = __builtin_ldexpf(1.0f, Mma<CODEC>::kCodeShift - Mma<CODEC>::kWeightTop);
  const float sum = l + other_half(l);
  const int64_t rh = static_cast<int64_t>(tile.first + row_i) * a.heads + head * group + row_h;
  if (a.splits > 1) {
    const int64_t per_part = c.rows * c.heads, part = split * per_part + rh;
    if (h == 0) {
      part_ml(c, part)[0] = m;
      part_ml(c, part)[1] = sum;
    }
    if (sum == 0.0f) return;
    float* o = part_acc(c, a.splits * per_part, part);
#pragma unroll
    for (int i = 0; i < HDP / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 32 * i + 8 * (r >> 2) + 4 * h + (r & 3);
        if (EXACT || d < a.hd) o[d] = acc[i][r] * back;
      }
    return;
  }
  if (c.lse != nullptr && h == 0) c.lse[rh] = sum == 0.0f ? -__builtin_inff() : (m + log2f(sum)) * kLn2;
  const float over = sum == 0.0f ? 0.0f : back / sum;
#pragma unroll
  for (int i = 0; i < HDP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * i + 2 * r + 4 * h;
      if constexpr (EXACT) {
        uint32_t o[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float v0 = sum == 0.0f ? 0.0f : acc[i][r + 2 * e] * over, v1 = sum == 0.0f ? 0.0f : acc[i][r + 2 * e + 1] * over;
          o[e] = (f32_to_lin<DT>(v0) & 0xFFFFu) | f32_to_lin<DT>(v1) << 16;
        }
        uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(c.out) + rh * HDP + d);
        to[0] = o[0];
        to[1] = o[1];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < a.hd) store_o<DT>(c.out, rh * a.hd + d + e, sum == 0.0f ? 0.0f : acc[i][r + e] * over);
      }
    }
}

template <int HDP, bool EXACT, int CODEC, int DT>
hipError_t launch_as(const AttnCall& c, hipStream_t stream) {
  const RowsArgs a = rows_args(c, kWideRows);
  int64_t tiles = tiles_bound(c, kWideRows);
  if (tiles < 1) tiles = 1;  // rows of no sequence are still to be filled
  const int64_t groups = tiles * c.kv_heads * c.splits;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_wide_kernel<HDP, EXACT, CODEC, DT>), dim3(static_cast<uint32_t>(groups)),
                     dim3(kBlockThreads), 0, stream, a, static_cast<uint32_t>(tiles));
  return hipGetLastError();
}

template <int CODEC, int DT>
hipError_t launch_typed(const AttnCall& c, hipStream_t stream) {
  // Whole rows of 64 or 128 dims whose queries can be read by 16 and outputs written by 4 bytes.
  const bool whole = reinterpret_cast<uint64_t>(c.query) % 16 == 0 && c.query_row_stride % 8 == 0 &&
                     c.query_head_stride % 8 == 0 && reinterpret_cast<uint64_t>(c.out) % 4 == 0;
  if (c.head_dim == 64 && whole) return launch_as<64, true, CODEC, DT>(c, stream);
  if (c.head_dim <= 64) return launch_as<64, false, CODEC, DT>(c, stream);
  if (c.head_dim == 128 && whole) return launch_as<128, true, CODEC, DT>(c, stream);
  return launch_as<128, false, CODEC, DT>(c, stream);
}

}  // namespace

hipError_t launch_wide(const AttnCall& c, hipStream_t stream) {
  if (c.dtype == kLinF16)
    return c.codec == kE4M3 ? launch_typed<kE4M3, kLinF16>(c, stream) : launch_typed<kE5M2, kLinF16>(c, stream);
  return c.codec == kE4M3 ? launch_typed<kE4M3, kLinBF16>(c, stream) : launch_typed<kE5M2, kLinBF16>(c, stream);
}

}  // namespace attn
}  // namespace kvhip
