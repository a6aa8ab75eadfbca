// Shared by the matrix-core forms over paged caches of 16-bit values: products, units of 8 tokens and their table
// entries, the transposition of K, and the way back to float32 for rows whose sums are no finite numbers.
#pragma once

#include <type_traits>

#include "kv_cache_attention.h"

namespace kvhip {
namespace catt {

template <int DT>
struct Mma16;

template <>
struct Mma16<kLinF16> {
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
struct Mma16<kLinBF16> {
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

constexpr int kTilePlaces = 128;  // places of a wave's tile, 16 units of 8

// Table column of a position.  (block_shift is log2(block_size) here, or -1.)
__device__ __forceinline__ uint32_t block_column(const CacheArgs& a, int32_t token) {
  return a.r.block_shift >= 0 ? static_cast<uint32_t>(token) >> a.r.block_shift
                              : static_cast<uint32_t>(token) / static_cast<uint32_t>(a.r.bs);
}

// Byte offset of a block's place from its cache's beginning: strides are below 2^32 (see tiles_fit).
__device__ __forceinline__ uint64_t block_offset(const CacheArgs& a, int kv, int32_t block, int32_t place) {
  return static_cast<uint64_t>(static_cast<uint32_t>(block)) * static_cast<uint32_t>(a.r.c.cache_block_stride[kv]) +
         static_cast<uint32_t>(2 * place);
}

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
  const uint32_t lo = __shfl(static_cast<uint32_t>(v), lane), hi = __shfl(static_cast<uint32_t>(v >> 32), lane);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// Maximum and sum over the four lane groups of 16, without LDS: the swaps leave both halves of what they exchange.
__device__ __forceinline__ float four_max(float v) {
  const u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a.x), __uint_as_float(a.y));
  const u32x2 b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b.x), __uint_as_float(b.y));
}

// How far (in powers of two) a row's maximum may pass the reference its weights are taken to before sums so far are
// scaled to a new one: float16 weights of up to 2^15 fit, for the others there is much room.
template <int DT>
constexpr float kSlack = DT == kLinF16 ? 1.0f : 8.0f;

// The table entry of the unit of 8 places from v on, on its way (see load_entry for the FP8 caches).
struct UnitEntry {
  uint32_t lo, hi;
};

__device__ __forceinline__ UnitEntry load_unit(const CacheArgs& a, const View& w, const uint8_t* table, int32_t v,
                                               int32_t end) {
  if (end <= 0) return {0xFFFFFFFFu, 0xFFFFFFFFu};
  const uint32_t column = block_column(a, position(w, min(v, (end - 1) & ~7)));
  const uint8_t* p = table + static_cast<uint64_t>(column) * (a.r.c.wide_tables ? 8 : 4);
  return {load4(p), load4(p + (a.r.c.wide_tables ? 4 : 0))};
}

// A unit: its block and place there (those of block 0 where it has none, which is always there to be read), and which
// of its tokens any row of the tile sees.
struct Unit {
  int32_t block, place;
  uint32_t bits;
};

__device__ __forceinline__ Unit resolve_unit(const CacheArgs& a, const View& w, const UnitEntry& e, int32_t v, int32_t end) {
  const bool good = v < end && e.lo < static_cast<uint32_t>(a.r.num_blocks) && (!a.r.c.wide_tables || e.hi == 0);
  if (!good) return {0, 0, 0};
  const int32_t token = position(w, v);
  const int32_t place = a.r.block_shift >= 0 ? token & (a.r.bs - 1)
                                             : token - static_cast<int32_t>(block_column(a, token)) * a.r.bs;
  return {static_cast<int32_t>(e.lo), place, tile_bits(w, token)};
}

// Whether every row of the tile sees all of the `places` places from v on, as far as the rows themselves go.
__device__ __forceinline__ bool all_rows_see(const CacheArgs& a, const View& w, int32_t v, int places) {
  if (v < w.front) return false;
  const int32_t from = v + w.gap, last = from + places - 1;
  if (a.masks != nullptr) return last < w.before;
  return last <= w.pos_lo && (a.window == 0 || from > w.pos_hi - a.window);
}

// Token t of the 8 rows' 16 bytes: 8 dims, as an operand of the product.
__device__ __forceinline__ u32x4 token_dims(const u32x4 (&raw)[8], int t) {
  u32x4 out;
#pragma unroll
  for (int p = 0; p < 4; ++p)
    out[p] = __builtin_amdgcn_perm(raw[2 * p + 1][t >> 1], raw[2 * p][t >> 1], (t & 1) != 0 ? 0x07060302u : 0x05040100u);
  return out;
}

// Ones in the halves of the tokens whose bits are set.
__device__ __forceinline__ u32x4 token_masks(uint32_t bits) {
  u32x4 out;
#pragma unroll
  for (int p = 0; p < 4; ++p)
    out[p] = ((bits >> (2 * p) & 1u) != 0 ? 0xFFFFu : 0u) | ((bits >> (2 * p + 1) & 1u) != 0 ? 0xFFFF0000u : 0u);
  return out;
}

__device__ __forceinline__ const uint8_t* stepped(const uint8_t* p) {
  asm volatile("" : "+v"(p));
  return p;
}

// Row and head of the in_tile-th row of a tile.
struct TilePlace {
  int64_t row, head;
};

__device__ __forceinline__ TilePlace tile_place(const CacheArgs& a, const RowTile& tile, int32_t kv_head, int32_t in_tile) {
  const int32_t at = tile.base + in_tile;
  const int32_t i = at / a.r.group;
  return {static_cast<int64_t>(tile.first) + i, static_cast<int64_t>(kv_head) * a.r.group + (at - i * a.r.group)};
}

// The tile's queries in LDS as the products read them: for 16 rows and 32 dims, lane (x, g) has row x with the dims
// 32 k + 4 i + g, i = 0..7.
template <int DT, int HD, int NT>
__device__ __forceinline__ void stage_queries(const CacheArgs& a, const RowTile& tile, int32_t kv_head, int32_t tile_rows,
                                              u32x4* queries) {
  const AttnCall& c = a.r.c;
  const uint16_t* from = static_cast<const uint16_t*>(c.query);
  uint16_t* to = reinterpret_cast<uint16_t*>(queries);
  auto place = [](int row, int d) {
    const int lane = (d & 3) * 16 + (row & 15), i = (d & 31) >> 2;
    return (((row >> 4) * (HD / 32) + d / 32) * kWave + lane) * 8 + i;
  };
  auto row_of = [&](int row) {
    const TilePlace p = tile_place(a, tile, kv_head, row);
    return from + p.row * c.query_row_stride + p.head * c.query_head_stride;
  };
  if (((reinterpret_cast<uint64_t>(from) | 2 * c.query_row_stride | 2 * c.query_head_stride) & 15) == 0) {
#pragma unroll 4
    for (int at = threadIdx.x; at < 16 * NT * HD / 8; at += kBlockThreads) {
      const int row = at / (HD / 8), d = at % (HD / 8) * 8;
      u32x4 dims{};
      if (row < tile_rows) dims = ld16_cached(reinterpret_cast<const uint8_t*>(row_of(row) + d));
#pragma unroll
      for (int k = 0; k < 8; ++k) to[place(row, d + k)] = static_cast<uint16_t>(elem16(dims, k));
    }
    return;
  }
  for (int at = threadIdx.x; at < 16 * NT * HD; at += kBlockThreads) {
    const int row = at / HD, d = at % HD;
    to[place(row, d)] = row < tile_rows ? row_of(row)[d] : 0;
  }
}

template <int DT>
__device__ __forceinline__ void store4(void* base, int64_t at, f32x4 o) {
  u32x2 v;
  v.x = pack16(f32_to_lin<DT>(o.x), f32_to_lin<DT>(o.y));
  v.y = pack16(f32_to_lin<DT>(o.z), f32_to_lin<DT>(o.w));
  *reinterpret_cast<KVHIP_GLOBAL u32x2*>(reinterpret_cast<uint64_t>(static_cast<uint16_t*>(base) + at)) = v;
}

// Rows whose sums are infinite or no numbers, once more without matrix products.  A weight of 0 times an infinite or
// NaN value of a position that this row does not see, but another of the tile does, is what makes most of them, since a
// product cannot leave a value out; sums over bf16's largest values are the others.  rows: bits of the rows from
// first_row of the tile on; scratch: LDS that nothing else uses any more.
template <int DT, int HD>
__device__ __forceinline__ void redo_rows(const CacheArgs& a, const View& w, const RowTile& tile, int32_t kv_head,
                                          int64_t line, int32_t part, int32_t count, int32_t lo, int32_t hi,
                                          uint32_t rows, int32_t first_row, float* scratch) {
  const AttnCall& c = a.r.c;
  const int lane = lane_id(), wave = wave_in_block();
  constexpr int kFloats = HD + (sizeof(VisitScratch) + 15) / 16 * 4;
  float* q = scratch + wave * kFloats;
  VisitScratch& visit = *reinterpret_cast<VisitScratch*>(q + HD);
  for (int32_t turn = 0; rows != 0; rows &= rows - 1, ++turn) {
    if (turn % kWavesPerBlock != wave) continue;
    const int32_t in_tile = first_row + __builtin_ctz(rows);
    const TilePlace p = tile_place(a, tile, kv_head, in_tile);
    for (int d = lane; d < HD; d += kWave)
      q[d] = load_q<DT>(c.query, p.row * c.query_row_stride + p.head * c.query_head_stride + d);
    __builtin_amdgcn_wave_barrier();
    constexpr int kMine = (HD + kWave - 1) / kWave;
    float m = 0.0f, l = 0.0f, out[kMine] = {};
    const RowSight sight = row_sight(a, w, tile.first, static_cast<int32_t>(p.row) - tile.first);
    for (float lower = 0.0f;; lower = kLower) {
      float top, sum, acc[kMine];
      visit_row<DT, kMine * kWave>(a, w, tile.seq, sight, kv_head, q, lo, hi, kWave, lower, visit, top, sum, acc);
      bool over = false;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (lower == 0.0f || !__builtin_isfinite(out[i])) out[i] = sum == 0.0f ? 0.0f : acc[i] / sum;
        over |= !__builtin_isfinite(out[i]);
      }
      if (lower == 0.0f) {
        m = top;
        l = sum;
      }
      if (DT == kLinF16 || lower != 0.0f || !__builtin_isfinite(sum) || ballot(over) == 0) break;
    }
    const int64_t slot = slot_row(a, line, part, in_tile);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int d = lane + i * kWave;
      if (d >= HD) continue;
      if (count > 1) slot_out(a, slot)[d] = out[i];
      else store_o<DT>(c.out, (p.row * c.heads + p.head) * HD + d, out[i]);
    }
    if (lane == 0) {
      if (count > 1) {
        slot_ml(a, slot)[0] = m;
        slot_ml(a, slot)[1] = l;
      } else if (c.lse != nullptr) {
        c.lse[p.row * c.heads + p.head] = log_sum(m, l);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// kv_cache_attention_rows.hip: tiles of 16 * nt rows.
hipError_t launch_rows(const CacheArgs& a, int nt, hipStream_t stream);

// kv_cache_attention_wide.hip: tiles of kWideTileRows rows.
constexpr int kWideTileRows = 128;
hipError_t launch_wide_tiles(const CacheArgs& a, hipStream_t stream);

}  // namespace catt
}  // namespace kvhip
