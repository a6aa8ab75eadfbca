// Attention over paged caches of 16-bit values: the form for many rows (prompt chunks, wide trees).
//
// A workgroup takes 128 rows of one sequence and one part of the positions, 64 positions at a time: a tile of K and V is
// brought into LDS once, as the operands of the products, and read by its four waves, 32 rows each.
//   * Product j of S^T = K Q^T (j = 0..3) has in its row 4 g + r the token 4 (j % 2) + r of unit 4 (j / 2) + g, a unit
//     being 8 positions: lane (x, g) then has, of row x, all 8 tokens of unit 4 h + g in products 2 h and 2 h + 1, which
//     is what the product with V's 16 bytes of that unit takes.
//   * K is brought in by lanes that each read 4 rows of 16 bytes, d = 32 k + 16 h + 4 i + g, i = 0..3 (four rows of a
//     block, a 128-byte line, in an instruction), and turned with byte permutes into 4 dims of each of the 8 tokens.
// The next tile's loads are on their way while a tile is worked on, in registers; two tiles of LDS leave one barrier a
// tile.  A weight goes in as two summands of the caches' type, as in the form for few rows: rounded once, a row's output
// would be off by 2^-8 of its values (bf16), and by how much would go with the form that its neighbours in the call bring
// about.  Bound by vector instructions (about nine for a score, one of them an exponential of a quarter of the rate) next to
// the matrix ones: matrix units busy 35 % of the time, vector ones 49 %, 1.6 waves a SIMD on average.  Chunks of 1753 and
// 2048 rows with a window of 4000 (32 heads, 8 in the cache, 128 dims, bf16): 434 us, 575 TFLOP/s without the second
// products; with one summand 329.
#include "kv_cache_attention_tiles.h"

namespace kvhip {
namespace catt {
namespace {

constexpr int kWideTile = 64;  // positions
constexpr int kWaveRows = kWideTileRows / kWavesPerBlock;
constexpr int kReads = 4;  // operands on their way from LDS

template <int HD>
struct WideTile {  // 1 KiB of 64 lanes for each operand
  u32x4 keys[4][HD / 32][kWave];    // product, step of 32 dims
  u32x4 values[2][HD / 16][kWave];  // half of the units, 16 dims
};

template <int DT, int HD>
__global__ __launch_bounds__(kBlockThreads, 2) void cache_wide_kernel(const CacheArgs a) {
  constexpr int kSteps = HD / 32, kDimTiles = HD / 16;
  constexpr int kMyKeys = (kSteps + kWavesPerBlock - 1) / kWavesPerBlock, kMyValues = 2 * kDimTiles / kWavesPerBlock;
  static_assert(2 * kDimTiles % kWavesPerBlock == 0, "values are dealt out evenly");
  const AttnCall& c = a.r.c;
  const int lane = lane_id(), wave = wave_in_block(), x = lane & 15, g = lane >> 4;
  // Neighbours in the launch are the kv heads of a row tile, and go to different XCDs: with 8 of them a head's tiles
  // meet in one L2.  Later tiles see more, and come first.
  const int32_t kv_head = blockIdx.x % static_cast<uint32_t>(c.kv_heads);
  const int32_t index = a.tiles - 1 - static_cast<int32_t>(blockIdx.x / static_cast<uint32_t>(c.kv_heads));
  const int32_t part = blockIdx.y;
  const int64_t line = static_cast<int64_t>(index) * c.kv_heads + kv_head;
  __shared__ WideTile<HD> tiles[2];
  __shared__ uint32_t odd_rows[kWavesPerBlock];

  if (part == 0 && c.starts != nullptr && writes_loose_rows(c))
    fill_loose_rows<DT>(c, index, a.tiles, kv_head * a.r.group, a.r.group);
  const RowTile tile = find_tile(a.r, index, kWideTileRows);
  View w{};
  int32_t count = 0;
  if (tile.seq >= 0) {
    w = tile_view(a, tile, kWideTileRows);
    count = part_count(a, w.length);
  }
  if (part == 0 && threadIdx.x == 0 && a.parts > 1) *line_of(a, line) = Line{count, tile.first, tile.count, tile.base};
  if (part >= count) return;
  const Span span = part_places(a, w.length, part, count);
  const int32_t lo = static_cast<int32_t>(span.lo), hi = static_cast<int32_t>(span.hi);
  const int32_t tile_rows = min(kWideTileRows, tile.count * a.r.group - tile.base);
  if (threadIdx.x < kWavesPerBlock) odd_rows[threadIdx.x] = 0;

  const uint8_t* table = static_cast<const uint8_t*>(c.tables) +
                         static_cast<int64_t>(tile.seq) * c.table_stride * (c.wide_tables ? 8 : 4);
  // Lane: units, halves of 32 dims and quarters of those, so that the 8 bytes that 32 lanes write to LDS at a time lie on
  // different banks.  Unit k is in lane 32 (k / 4) + k % 4.
  const int32_t my_unit8 = 8 * ((lane & 3) | lane >> 5 << 2);
  UnitEntry entry = load_unit(a, w, table, lo + my_unit8, hi);

  // Each wave's queries, by way of LDS.
  u32x4 query[2][kSteps];
  {
    u32x4* staged = reinterpret_cast<u32x4*>(&tiles[0]);
    static_assert(sizeof(tiles) >= sizeof(u32x4) * (kWideTileRows / 16) * kSteps * kWave, "the queries fit the tiles");
    stage_queries<DT, HD, kWideTileRows / 16>(a, tile, kv_head, tile_rows, staged);
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) query[nt][ks] = staged[((2 * wave + nt) * kSteps + ks) * kWave + lane];
    __syncthreads();
  }

  RowSight sight[2];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    const int32_t at = min(tile.base + kWaveRows * wave + 16 * nt + x, tile.count * a.r.group - 1);
    sight[nt] = row_sight(a, w, tile.first, at / a.r.group);
  }
  // The wave's first and last position, for the tiles that all its rows see.
  View mine = w;
  mine.pos_lo = w.before + min(tile.base + kWaveRows * wave, tile.count * a.r.group - 1) / a.r.group;
  mine.pos_hi = w.before + min(tile.base + kWaveRows * wave + kWaveRows - 1, tile.count * a.r.group - 1) / a.r.group;
  float m[2], l[2];
  f32x4 acc[2][kDimTiles];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    m[nt] = -__builtin_inff();
    l[nt] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt) acc[nt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const int64_t row_bytes = static_cast<int64_t>(a.r.bs) * 2;
  const int key_g = lane >> 3 & 3, key_half = lane >> 2 & 1;
  const int key_slot = 16 * g + (x ^ g);
  const uint8_t* key = static_cast<const uint8_t*>(c.cache[0]) +
                       (static_cast<int64_t>(kv_head) * HD + 16 * key_half + key_g) * row_bytes;
  const uint8_t* value = static_cast<const uint8_t*>(c.cache[1]) + (static_cast<int64_t>(kv_head) * HD + x) * row_bytes;
  u32x4 raw_keys[kMyKeys][4], raw_values[kMyValues];
  // The lane's shares of a tile: step wave + 4 n of K, image wave + 4 n of V (dims of 16, then the half of the units).
  auto load_tile = [&](const Unit& unit) {
    const uint8_t* k = key + block_offset(a, 0, unit.block, unit.place);
    const uint64_t v = block_offset(a, 1, unit.block, unit.place);
#pragma unroll
    for (int n = 0; n < kMyKeys; ++n) {
      if (kSteps % kWavesPerBlock != 0 && wave + kWavesPerBlock * n >= kSteps) break;
      const uint8_t* from = k + 32 * (wave + kWavesPerBlock * n) * row_bytes;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        raw_keys[n][i] = ld16_cached(from);
        from = stepped(from + 4 * row_bytes);
      }
    }
#pragma unroll
    for (int n = 0; n < kMyValues; ++n) {
      const int image = wave + kWavesPerBlock * n, half = image / kDimTiles, dt = image % kDimTiles;
      raw_values[n] = ld16_cached(value + 16 * dt * row_bytes + shfl64(v, 32 * half + g));
    }
  };
  auto store_tile = [&](WideTile<HD>& to, const Unit& unit, bool masked) {
#pragma unroll
    for (int n = 0; n < kMyKeys; ++n) {
      const int ks = wave + kWavesPerBlock * n;
      if (kSteps % kWavesPerBlock != 0 && ks >= kSteps) break;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        u32x2 dims;
#pragma unroll
        for (int p = 0; p < 2; ++p)
          dims[p] = __builtin_amdgcn_perm(raw_keys[n][2 * p + 1][t >> 1], raw_keys[n][2 * p][t >> 1],
                                          (t & 1) != 0 ? 0x07060302u : 0x05040100u);
        // Unit u is 4 (j / 2) + g of product j = 2 (u / 4) + t / 4, its token t in row 4 (u % 4) + t % 4.
        const int j = 2 * (lane >> 5) + (t >> 2), row = 4 * (lane & 3) + (t & 3);
        reinterpret_cast<u32x2*>(&to.keys[j][ks][16 * key_g + (row ^ key_g)])[key_half] = dims;
      }
    }
#pragma unroll
    for (int n = 0; n < kMyValues; ++n) {
      const int image = wave + kWavesPerBlock * n, half = image / kDimTiles, dt = image % kDimTiles;
      if (masked) raw_values[n] &= token_masks(__shfl(unit.bits, 32 * half + g));
      to.values[half][dt][lane] = raw_values[n];
    }
  };

  Unit unit = resolve_unit(a, w, entry, lo + my_unit8, hi);
  entry = load_unit(a, w, table, lo + kWideTile + my_unit8, hi);
  if (lo < hi) {
    load_tile(unit);
    store_tile(tiles[0], unit, ballot(unit.bits != 0xFFu) != 0);
  }
  __syncthreads();
  int turn = 0;
  for (int32_t v0 = lo; v0 < hi; v0 += kWideTile, turn ^= 1) {
    const WideTile<HD>& at = tiles[turn];
    const Unit next = resolve_unit(a, w, entry, v0 + kWideTile + my_unit8, hi);
    entry = load_unit(a, w, table, v0 + 2 * kWideTile + my_unit8, hi);
    const bool masked = ballot(unit.bits != 0xFFu) != 0 || !all_rows_see(a, mine, v0, kWideTile);

    f32x4 s[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[nt][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // Operands are read from LDS kReads ahead; left alone, the compiler waits for each before it asks for the next.
    u32x4 operand[kReads];
#pragma unroll
    for (int n = 0; n < kReads; ++n) operand[n] = at.keys[n & 3][n >> 2][key_slot];
#pragma unroll
    for (int n = 0; n < 4 * kSteps; ++n) {
      const int ks = n >> 2, j = n & 3;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) s[nt][j] = Mma16<DT>::mma(operand[n % kReads], query[nt][ks], s[nt][j]);
      if (n + kReads < 4 * kSteps) operand[n % kReads] = at.keys[(n + kReads) & 3][(n + kReads) >> 2][key_slot];
      __builtin_amdgcn_sched_barrier(0);
    }
    if (masked) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t bits = __shfl(unit.bits, 32 * half + g);
        const int32_t token = position(w, v0 + 8 * (4 * half + g));
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const uint32_t seen = bits & row_bits(a, w, sight[nt], token);
#pragma unroll
          for (int t = 0; t < 8; ++t)
            if ((seen >> t & 1u) == 0) s[nt][2 * half + (t >> 2)][t & 3] = -__builtin_inff();
        }
      }
    }
    load_tile(next);
    // The factor is positive here: the largest product is the largest score's.
    float top[2];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      float most = s[nt][0][0];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = fmaxf(most, s[nt][j][r]);
      top[nt] = __builtin_fmaf(four_max(most), a.factor, -kTop<DT>);
    }
    if (ballot(top[0] > m[0] + kSlack<DT> || top[1] > m[1] + kSlack<DT>) != 0) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        top[nt] = fmaxf(m[nt], top[nt]);
        const float fade = fade_to(m[nt], top[nt]);
        l[nt] *= fade;
#pragma unroll
        for (int dt = 0; dt < kDimTiles; ++dt) acc[nt][dt] *= fade;
        m[nt] = top[nt];
      }
    }
    u32x4 weight[2][2][2];  // half, row tile, summand
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const float ref = m[nt] == -__builtin_inff() ? 0.0f : m[nt];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nt][j][r], a.factor, -ref));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nt][j][r + 1], a.factor, -ref));
          l[nt] += p0 + p1;
          const uint32_t high = Mma16<DT>::pack(p0, p1);
          const f32x2 back = Mma16<DT>::unpack(high);
          weight[j >> 1][nt][0][2 * (j & 1) + (r >> 1)] = high;
          weight[j >> 1][nt][1][2 * (j & 1) + (r >> 1)] = Mma16<DT>::pack(p0 - back.x, p1 - back.y);
        }
    }
#pragma unroll
    for (int n = 0; n < kReads; ++n) operand[n] = at.values[0][n][lane];
    __builtin_amdgcn_sched_barrier(0);  // the sums above are made here, not carried on as 32 summands
#pragma unroll
    for (int n = 0; n < 2 * kDimTiles; ++n) {
      const int half = n / kDimTiles, dt = n % kDimTiles;
#pragma unroll
      for (int summand = 0; summand < 2; ++summand)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
          acc[nt][dt] = Mma16<DT>::mma(operand[n % kReads], weight[half][nt][summand], acc[nt][dt]);
      if (n + kReads < 2 * kDimTiles)
        operand[n % kReads] = at.values[(n + kReads) / kDimTiles][(n + kReads) % kDimTiles][lane];
      __builtin_amdgcn_sched_barrier(0);
    }
    // (Behind the last tile: block 0, which is not looked at.)
    store_tile(tiles[turn ^ 1], next, ballot(next.bits != 0xFFu) != 0);
    unit = next;
    __syncthreads();
  }

#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    const float sum = groups_sum(l[nt]);
    const int32_t in_tile = kWaveRows * wave + 16 * nt + x;
    bool odd = !__builtin_isfinite(sum);
    if (in_tile < tile_rows) {
      const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
      const TilePlace to = tile_place(a, tile, kv_head, in_tile);
      const int64_t slot = slot_row(a, line, part, in_tile);
#pragma unroll
      for (int dt = 0; dt < kDimTiles; ++dt) {
        const f32x4 o = acc[nt][dt];
        odd |= !__builtin_isfinite(o.x + o.y + o.z + o.w);
        if (count > 1) *reinterpret_cast<f32x4*>(slot_out(a, slot) + 16 * dt + 4 * g) = o * scale;
        else store4<DT>(c.out, (to.row * c.heads + to.head) * HD + 16 * dt + 4 * g, o * scale);
      }
      if (g == 0) {
        if (count > 1) {
          slot_ml(a, slot)[0] = m[nt];
          slot_ml(a, slot)[1] = sum;
        } else if (c.lse != nullptr) {
          c.lse[to.row * c.heads + to.head] = log_sum(m[nt], sum);
        }
      }
      if (odd) atomicOr(&odd_rows[wave], 1u << (16 * nt + x));
    }
  }
  __syncthreads();
  for (int k = 0; k < kWavesPerBlock; ++k)
    if (odd_rows[k] != 0)
      redo_rows<DT, HD>(a, w, tile, kv_head, line, part, count, lo, hi, odd_rows[k], kWaveRows * k,
                        reinterpret_cast<float*>(&tiles[0]));
}

template <int DT>
hipError_t launch_dt(const CacheArgs& a, dim3 grid, hipStream_t stream) {
  switch (a.r.hd) {
    case 64: cache_wide_kernel<DT, 64><<<grid, kBlockThreads, 0, stream>>>(a); break;
    case 96: cache_wide_kernel<DT, 96><<<grid, kBlockThreads, 0, stream>>>(a); break;
    default: cache_wide_kernel<DT, 128><<<grid, kBlockThreads, 0, stream>>>(a); break;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_wide_tiles(const CacheArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(a.lines), a.parts);
  return a.r.c.dtype == kLinF16 ? launch_dt<kLinF16>(a, grid, stream) : launch_dt<kLinBF16>(a, grid, stream);
}

}  // namespace catt
}  // namespace kvhip
