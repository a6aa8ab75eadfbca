// Attention over paged caches of 16-bit values: the form for few rows (decode steps, drafts, small trees).
//
// A workgroup takes 16 * NT rows (a row is a position and a head of the kv head's group) of one sequence and one part
// of the positions; its four waves take 128 positions at a time in turn.  S^T = K Q^T, then O^T += V^T P^T, with
// 16x16x32 matrix instructions whose operands come straight from the cache's layout [head_dim][tokens of a block]:
//   * The 128 positions are 16 units of 8.  K: lane (x, g), x = lane % 16, g = lane / 16, loads 16 bytes, the 8 tokens
//     of unit s(x), of the rows d = 32 k + 4 i + g: an instruction takes 4 whole rows of each unit, a 128-byte line of
//     every block of 16 tokens.  The dwords of 8 rows i hold two tokens each; one byte permute of two rows makes a dword
//     of two dims, so eight products (one per token of the units) cover the tile, with the query's dims in the same
//     order.
//   * Their results give lane (x, g) the scores of row x with the 8 tokens of the units s(4 g + r), r = 0..3.  As the
//     second operand of V^T P^T these are 8 neighbours along the tokens, as 16 bytes of V are: lane (x, g) loads those
//     of dim 16 l + x.  No value crosses lanes but the running maximum.
//   * s(4 g + r) = 8 (g / 2) + 2 r + g % 2: the units of lanes g = 0, 1 (and 2, 3) are the halves of one block.
// The path is bound by the reads of K and V; the products of 16 rows take a twentieth of their time, and so weights may go
// in as two summands of the caches' type (a rounding of 2^-16 and less), which costs half as many products again.  48
// decode rows of 295 to 8192 tokens (32 heads, 8 of them in the cache, 128 dims, bf16): 176 to 191 us with the join, by
// where the caches lie, 4.2 to 4.6 TB/s.
// With each group of loads asked for where it is used it was 326.
#include "kv_cache_attention_tiles.h"

namespace kvhip {
namespace catt {
namespace {

template <int NT>
constexpr int kRowsOf = 16 * NT;

template <int DT, int HD, int NT>
__global__ __launch_bounds__(kBlockThreads, 2) void cache_rows_kernel(const CacheArgs a) {
  constexpr int kSteps = HD / 32, kDimTiles = HD / 16, kRows = kRowsOf<NT>;
  constexpr int kPitch = HD + 4;  // floats between the rows of the exchange: 16 rows on different banks
  const AttnCall& c = a.r.c;
  const int lane = lane_id(), wave = wave_in_block(), x = lane & 15, g = lane >> 4;
  const int32_t kv_head = blockIdx.y, part = blockIdx.z;
  const int64_t line = static_cast<int64_t>(blockIdx.x) * c.kv_heads + kv_head;
  __shared__ u32x4 queries[NT * kSteps * kWave];
  __shared__ __attribute__((aligned(16))) float exchange[kWavesPerBlock][16 * kPitch];
  __shared__ float ml_of[kWavesPerBlock][kRows][2];
  __shared__ uint32_t odd_rows;

  if (part == 0 && c.starts != nullptr && writes_loose_rows(c))
    fill_loose_rows<DT>(c, blockIdx.x, gridDim.x, kv_head * a.r.group, a.r.group);
  const RowTile tile = find_tile(a.r, blockIdx.x, kRows);
  View w{};
  int32_t count = 0;
  if (tile.seq >= 0) {
    w = tile_view(a, tile, kRows);
    count = part_count(a, w.length);
  }
  if (part == 0 && threadIdx.x == 0 && a.parts > 1) *line_of(a, line) = Line{count, tile.first, tile.count, tile.base};
  if (part >= count) return;
  const Span span = part_places(a, w.length, part, count);
  const int32_t lo = static_cast<int32_t>(span.lo), hi = static_cast<int32_t>(span.hi);
  const int32_t tile_rows = min(kRows, tile.count * a.r.group - tile.base);

  const uint8_t* table = static_cast<const uint8_t*>(c.tables) +
                         static_cast<int64_t>(tile.seq) * c.table_stride * (c.wide_tables ? 8 : 4);
  const int32_t unit_k = 8 * (x >> 3) + 2 * (x & 3) + ((x >> 2) & 1);
  const int32_t unit_v = 8 * (g >> 1) + (g & 1);  // + 2 r
  int32_t v0 = lo + wave * kTilePlaces;
  UnitEntry entry = load_unit(a, w, table, v0 + 8 * unit_k, hi);

  stage_queries<DT, HD, NT>(a, tile, kv_head, tile_rows, queries);
  if (threadIdx.x == 0) odd_rows = 0;

  // Each lane's row of every 16: what it sees, its maximum and sum.
  RowSight sight[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int32_t at = min(tile.base + 16 * nt + x, tile.count * a.r.group - 1);
    sight[nt] = row_sight(a, w, tile.first, at / a.r.group);
  }
  float m[NT], l[NT];
  f32x4 acc[NT][kDimTiles];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -__builtin_inff();
    l[nt] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt) acc[nt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int64_t row_bytes = static_cast<int64_t>(a.r.bs) * 2;
  const uint8_t* key = static_cast<const uint8_t*>(c.cache[0]) + (static_cast<int64_t>(kv_head) * HD + g) * row_bytes;
  const uint8_t* value = static_cast<const uint8_t*>(c.cache[1]) + (static_cast<int64_t>(kv_head) * HD + x) * row_bytes;

  // Loads go in groups of 8 (8 KiB of the wave), one or two of them on their way at any time: kSteps of K, as many of V,
  // then the next tile's.
  u32x4 ahead[2][8];
  const uint8_t* k_unit;     // of the tile whose K is being loaded
  const uint8_t* v_unit[4];  // units r of the tile at hand
  // The addresses go on by steps, through `stepped`: the compiler would keep a register pair for each of the offsets.
  auto load_k = [&](int ks) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ahead[ks & 1][i] = ld16_cached(k_unit);
      k_unit = stepped(k_unit + 4 * row_bytes);
    }
  };
  auto load_v = [&](int group) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = (group * 8 + i) / kDimTiles;
      ahead[(kSteps + group) & 1][i] = ld16_cached(v_unit[r]);
      v_unit[r] = stepped(v_unit[r] + 16 * row_bytes);
    }
  };
  // masked: some row does not see some of the positions.  (Two copies of the body, with and without masks, spill.)
  auto one_tile = [&](bool masked, const Unit& unit, const Unit& next, bool more) {
    uint32_t bits[4];
    const uint64_t v_offset = block_offset(a, 1, unit.block, unit.place);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v_unit[r] = value + shfl64(v_offset, 4 * g + r);
      bits[r] = __shfl(unit.bits, 4 * g + r);
    }
    f32x4 s[NT][8];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int t = 0; t < 8; ++t) s[nt][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
      u32x4 q[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) q[nt] = queries[(nt * kSteps + ks) * kWave + lane];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const u32x4 tokens = token_dims(ahead[ks & 1], t);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][t] = Mma16<DT>::mma(tokens, q[nt], s[nt][t]);
      }
      if (ks + 2 < kSteps) load_k(ks + 2);
      else load_v(ks + 2 - kSteps);
      __builtin_amdgcn_sched_barrier(0);
    }
    k_unit = key + block_offset(a, 0, next.block, next.place);
    u32x4 weight[NT][2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int t = 0; t < 8; ++t) s[nt][t] *= a.factor;
      if (masked) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t seen = bits[r] & row_bits(a, w, sight[nt], position(w, v0 + 8 * (unit_v + 2 * r)));
#pragma unroll
          for (int t = 0; t < 8; ++t)
            if ((seen >> t & 1u) == 0) s[nt][t][r] = -__builtin_inff();
        }
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < 8; ++t) top = fmaxf(top, s[nt][t][r]);
      top = fmaxf(m[nt], four_max(top) - kTop<DT>);
      const float ref = top == -__builtin_inff() ? 0.0f : top;
      if (ballot(top != m[nt]) != 0) {
        const float fade = fade_to(m[nt], top);
        l[nt] *= fade;
#pragma unroll
        for (int dt = 0; dt < kDimTiles; ++dt) acc[nt][dt] *= fade;
        m[nt] = top;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < 8; t += 2) {
          const float p0 = __builtin_amdgcn_exp2f(s[nt][t][r] - ref), p1 = __builtin_amdgcn_exp2f(s[nt][t + 1][r] - ref);
          l[nt] += p0 + p1;
          const uint32_t high = Mma16<DT>::pack(p0, p1);
          const f32x2 back = Mma16<DT>::unpack(high);
          weight[nt][0][r][t / 2] = high;
          weight[nt][1][r][t / 2] = Mma16<DT>::pack(p0 - back.x, p1 - back.y);
        }
    }
#pragma unroll
    for (int group = 0; group < kSteps; ++group) {
      u32x4 (&values)[8] = ahead[(kSteps + group) & 1];
      if (masked) {  // what no row sees may be no number
#pragma unroll
        for (int i = 0; i < 8; ++i) values[i] &= token_masks(bits[(group * 8 + i) / kDimTiles]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = (group * 8 + i) / kDimTiles, dt = (group * 8 + i) % kDimTiles;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          acc[nt][dt] = Mma16<DT>::mma(values[i], weight[nt][0][r], acc[nt][dt]);
          acc[nt][dt] = Mma16<DT>::mma(values[i], weight[nt][1][r], acc[nt][dt]);
        }
      }
      if (group + 2 < kSteps) load_v(group + 2);
      else if (more) load_k(group + 2 - kSteps);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  Unit unit = resolve_unit(a, w, entry, v0 + 8 * unit_k, hi);
  entry = load_unit(a, w, table, v0 + kWavesPerBlock * kTilePlaces + 8 * unit_k, hi);
  if (v0 < hi) {
    k_unit = key + block_offset(a, 0, unit.block, unit.place);
    load_k(0);
    load_k(1);
  }
  __syncthreads();
  while (v0 < hi) {
    const int32_t v1 = v0 + kWavesPerBlock * kTilePlaces;
    const Unit next = resolve_unit(a, w, entry, v1 + 8 * unit_k, hi);
    entry = load_unit(a, w, table, v1 + kWavesPerBlock * kTilePlaces + 8 * unit_k, hi);
    one_tile(ballot(unit.bits != 0xFFu) != 0 || !all_rows_see(a, w, v0, kTilePlaces), unit, next, v1 < hi);
    unit = next;
    v0 = v1;
  }

  // The waves' sums, 16 rows at a time.
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] = groups_sum(l[nt]);
    if (g == 0) {
      ml_of[wave][16 * nt + x][0] = m[nt];
      ml_of[wave][16 * nt + x][1] = l[nt];
    }
  }
  const int32_t row16 = threadIdx.x >> 4, col = threadIdx.x & 15;  // 16 threads per row
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    __syncthreads();
    float top = -__builtin_inff();
    for (int k = 0; k < kWavesPerBlock; ++k) top = fmaxf(top, ml_of[k][16 * nt + x][0]);
    const float fade = fade_to(m[nt], top);
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt)
      *reinterpret_cast<f32x4*>(&exchange[wave][x * kPitch + 16 * dt + 4 * g]) = acc[nt][dt] * fade;
    __syncthreads();
    const int32_t in_tile = 16 * nt + row16;
    if (in_tile >= tile_rows) continue;
    float all_top = -__builtin_inff(), sum = 0.0f;
    for (int k = 0; k < kWavesPerBlock; ++k) all_top = fmaxf(all_top, ml_of[k][in_tile][0]);
    for (int k = 0; k < kWavesPerBlock; ++k) sum += ml_of[k][in_tile][1] * fade_to(ml_of[k][in_tile][0], all_top);
    const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
    const TilePlace to = tile_place(a, tile, kv_head, in_tile);
    const int64_t slot = slot_row(a, line, part, in_tile);
    bool odd = !__builtin_isfinite(sum);
#pragma unroll
    for (int j = 0; j < HD / 64; ++j) {
      const int32_t d = 4 * (col + 16 * j);
      f32x4 o = *reinterpret_cast<const f32x4*>(&exchange[0][row16 * kPitch + d]);
#pragma unroll
      for (int k = 1; k < kWavesPerBlock; ++k) o += *reinterpret_cast<const f32x4*>(&exchange[k][row16 * kPitch + d]);
      odd |= !__builtin_isfinite(o.x + o.y + o.z + o.w);
      if (count > 1) *reinterpret_cast<f32x4*>(slot_out(a, slot) + d) = o * scale;
      else store4<DT>(c.out, (to.row * c.heads + to.head) * HD + d, o * scale);
    }
    if constexpr (HD % 64 != 0) {
      const int32_t d = HD / 64 * 64 + 4 * col;
      if (d < HD) {
        f32x4 o = *reinterpret_cast<const f32x4*>(&exchange[0][row16 * kPitch + d]);
#pragma unroll
        for (int k = 1; k < kWavesPerBlock; ++k) o += *reinterpret_cast<const f32x4*>(&exchange[k][row16 * kPitch + d]);
        odd |= !__builtin_isfinite(o.x + o.y + o.z + o.w);
        if (count > 1) *reinterpret_cast<f32x4*>(slot_out(a, slot) + d) = o * scale;
        else store4<DT>(c.out, (to.row * c.heads + to.head) * HD + d, o * scale);
      }
    }
    if (odd) atomicOr(&odd_rows, 1u << in_tile);
    if (col == 0) {
      if (count > 1) {
        slot_ml(a, slot)[0] = all_top;
        slot_ml(a, slot)[1] = sum;
      } else if (c.lse != nullptr) {
        c.lse[to.row * c.heads + to.head] = log_sum(all_top, sum);
      }
    }
  }
  __syncthreads();
  if (odd_rows != 0)
    redo_rows<DT, HD>(a, w, tile, kv_head, line, part, count, lo, hi, odd_rows, 0, &exchange[0][0]);
}

template <int DT, int HD>
hipError_t launch_hd(const CacheArgs& a, dim3 grid, int nt, hipStream_t stream) {
  if constexpr (HD <= 128)
    if (nt == 2) {
      cache_rows_kernel<DT, HD, 2><<<grid, kBlockThreads, 0, stream>>>(a);
      return hipGetLastError();
    }
  cache_rows_kernel<DT, HD, 1><<<grid, kBlockThreads, 0, stream>>>(a);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_dt(const CacheArgs& a, dim3 grid, int nt, hipStream_t stream) {
  switch (a.r.hd) {
    case 64: return launch_hd<DT, 64>(a, grid, nt, stream);
    case 96: return launch_hd<DT, 96>(a, grid, nt, stream);
    case 128: return launch_hd<DT, 128>(a, grid, nt, stream);
    case 192: return launch_hd<DT, 192>(a, grid, nt, stream);
    default: return launch_hd<DT, 256>(a, grid, nt, stream);
  }
}

}  // namespace

hipError_t launch_rows(const CacheArgs& a, int nt, hipStream_t stream) {
  const dim3 grid(a.tiles, static_cast<uint32_t>(a.r.c.kv_heads), a.parts);
  return a.r.c.dtype == kLinF16 ? launch_dt<kLinF16>(a, grid, nt, stream) : launch_dt<kLinBF16>(a, grid, nt, stream);
}

}  // namespace catt
}  // namespace kvhip
