// The attention weight that cached tokens gather: kv_accumulate_attention_weights.
//
//   weights[b, h, j] += sum over the rows and heads of kv head h that see j of e^(s_j - lse)
//
// with the scores s_j of kv_cache_attention.hip and the logarithms it returned.  A token's sum is made by one
// workgroup, in the same order in every run: no atomics.
#include "kv_cache_attention_tiles.h"

namespace kvhip {
namespace catt {
namespace {

// Rows [first, end) of a sequence that can see one of the positions from .. last (places v0 and up).  Those in front of
// the first position see none of them; with a window, and no first tokens among them, those do not either whose window
// begins behind the last.
struct RowSpan {
  int32_t first, end;
};

__device__ __forceinline__ RowSpan rows_that_see(const CacheArgs& a, const View& w, int32_t count, int32_t v0,
                                                 int32_t from, int32_t last) {
  const bool past = a.window > 0 && v0 >= w.front && from >= a.sinks;
  return {min(max(from - w.before, 0), count), past ? min(max(last + a.window - w.before, 0), count) : count};
}

// ----- any shape and type: a thread per token, one row and head after the other --------------------
template <int DT>
__global__ __launch_bounds__(kBlockThreads) void weights_any_kernel(const CacheArgs a) {
  const AttnCall& c = a.r.c;
  const int32_t seq = blockIdx.y, head = blockIdx.z;
  const int64_t bs = a.r.bs, hd = a.r.hd;
  constexpr int64_t kElt = DT == kLinF32 ? 4 : 2;
  __shared__ float q[kVisitDims];
  const SeqRows rows = seq_rows(c, seq);
  if (rows.count == 0) return;
  const int32_t count = static_cast<int32_t>(rows.count);
  const View w = make_view(a, seq, count, 0, count - 1);
  for (int32_t base = blockIdx.x * kBlockThreads; base < w.length; base += gridDim.x * kBlockThreads) {
    const int32_t v = base + threadIdx.x;
    const int32_t token = position(w, v);
    int64_t k = -1;
    if (v < w.length && token < a.weight_tokens && (tile_bits(w, token) & 1u) != 0) {
      const int64_t blk = position_block(a, seq, token);
      if (blk >= 0) k = blk * (c.cache_block_stride[0] / kElt) + head * hd * bs + token % bs;
    }
    const RowSpan span = rows_that_see(a, w, count, base, base < w.front ? 0 : base + w.gap,
                                       position(w, base + kBlockThreads - 1));
    float sum = 0.0f;
    for (int32_t x = span.first * a.r.group; x < span.end * a.r.group; ++x) {
      const int32_t i = x / a.r.group;
      const int64_t row = rows.first + i, hq = head * a.r.group + x % a.r.group;
      __syncthreads();
      for (int64_t d = threadIdx.x; d < hd; d += kBlockThreads)
        q[d] = load_q<DT>(c.query, row * c.query_row_stride + hq * c.query_head_stride + d);
      __syncthreads();
      const float lse = c.lse[row * c.heads + hq];
      if (lse == -__builtin_inff() || k < 0 || (row_bits(a, w, row_sight(a, w, 0, i), token) & 1u) == 0) continue;
      float dot = 0.0f;
      for (int64_t d = 0; d < hd; ++d) dot = __builtin_fmaf(q[d], load_q<DT>(c.cache[0], k + d * bs), dot);
      // The difference first: it is small where a weight is large, and its product then loses nothing.
      float less = __builtin_fmaf(dot, a.scale, -lse);
      if (__builtin_isfinite(less)) less = __builtin_fmaf(dot, a.scale_rest, less);
      sum += __builtin_amdgcn_exp2f(less * kLog2e);
    }
    if (k >= 0) {
      float* to = a.weights + seq * a.weight_row_stride + head * a.weight_head_stride + token;
      *to += sum;
    }
  }
}

// ----- matrix-core form -----------------------------------------------------------------------------
// A wave keeps the keys of 128 positions (16 units of 8, see kv_cache_attention_rows.hip) as operands in registers and
// goes through the rows, 16 at a time: S^T = K Q^T.  Each lane adds up the weights that its row of every 16 gives its 32
// positions; the lanes' sums meet at the end.  Lane (x, g) holds the dims 32 k + 8 g + i of K here, so that 16 bytes of a
// query are an operand as they are.
// With few rows the waves of a workgroup take different positions (bound by the read of K: all of a wave's 32 loads are
// on their way at once), with many the same positions and a quarter of the rows each (bound by 32 exponentials of a
// quarter of the full rate next to 32 products).  16 decode rows of 430 to 4097 tokens: 20 us, 3.1 TB/s; chunks of 795 and
// 1024 rows over 3120 and 6001 tokens (32 heads, 8 in the cache, 128 dims): 116 us, 550 TFLOP/s; 4096 rows over as many
// tokens with a window of 64: 21 us, of 256: 30, without 144.
constexpr int kAtOnce = 4;     // tokens of the units whose scores are held at a time
constexpr int64_t kCus = 256;
// Row tiles of a sequence from which on the waves share positions: each of the four has one.
constexpr int kManyTiles = 4;

__device__ __forceinline__ float sum_of_16(float v) {  // over lanes that differ in x
#define KVHIP_ROTATE(n) \
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x120 + n, 0xF, 0xF, false))
  KVHIP_ROTATE(8);
  KVHIP_ROTATE(4);
  KVHIP_ROTATE(2);
  KVHIP_ROTATE(1);
#undef KVHIP_ROTATE
  return v;
}

template <int DT, int HD, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, HD <= 128 ? 2 : 1) void weights_tile_kernel(const CacheArgs a) {
  constexpr int kSteps = HD / 32;
  const AttnCall& c = a.r.c;
  const int lane = lane_id(), wave = wave_in_block(), x = lane & 15, g = lane >> 4;
  const int32_t seq = blockIdx.y, kv_head = blockIdx.z, group = a.r.group;
  __shared__ __attribute__((aligned(16))) float sums[WAVES][kTilePlaces];
  const SeqRows seq_rows_ = seq_rows(c, seq);
  if (seq_rows_.count == 0) return;
  const int32_t count = static_cast<int32_t>(seq_rows_.count), rows = count * group;
  const View w = make_view(a, seq, count, 0, count - 1);
  const bool many = a.parts > 1;  // the waves share positions
  const int32_t stride = many ? kTilePlaces : kTilePlaces * WAVES;
  const uint8_t* table = static_cast<const uint8_t*>(c.tables) +
                         static_cast<int64_t>(seq) * c.table_stride * (c.wide_tables ? 8 : 4);
  const int64_t row_bytes = static_cast<int64_t>(a.r.bs) * 2;
  const float* lse_of = c.lse + seq_rows_.first * c.heads + static_cast<int64_t>(kv_head) * group;
  const uint8_t* query = reinterpret_cast<const uint8_t*>(
      static_cast<const uint16_t*>(c.query) + seq_rows_.first * c.query_row_stride +
      static_cast<int64_t>(kv_head) * group * c.query_head_stride + 8 * g);
  const int group_log = (group & (group - 1)) == 0 ? __builtin_ctz(group) : -1;
  for (int32_t base = blockIdx.x * stride; base < w.length; base += gridDim.x * stride) {
    const int32_t v0 = base + (many ? 0 : wave * kTilePlaces);
    const UnitEntry entry = load_unit(a, w, table, v0 + 8 * x, w.length);
    const Unit unit = resolve_unit(a, w, entry, v0 + 8 * x, w.length);
    u32x4 keys[kSteps][8];
    {
      u32x4 raw[kSteps][8];
      const uint8_t* k = static_cast<const uint8_t*>(c.cache[0]) + block_offset(a, 0, unit.block, unit.place) +
                         (static_cast<int64_t>(kv_head) * HD + 8 * g) * row_bytes;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        const uint8_t* from = k;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          raw[ks][i] = ld16_cached(from);
          from = stepped(from + row_bytes);
        }
        k = stepped(k + 32 * row_bytes);
      }
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks)
#pragma unroll
        for (int t = 0; t < 8; ++t) keys[ks][t] = token_dims(raw[ks], t);
    }
    const bool whole = ballot(unit.bits != 0xFFu) == 0;
    // Positions of the tile: none of them is past last, none but first ones in front of from.
    const int32_t from = v0 < w.front ? 0 : v0 + w.gap, last = position(w, v0 + kTilePlaces - 1);
    f32x4 sum[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) sum[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    const int32_t step = many ? 16 * WAVES : 16;
    const RowSpan span = rows_that_see(a, w, count, v0, from, last);
    const int32_t end = __builtin_amdgcn_readfirstlane(v0 < w.length ? span.end * group : 0);
    int32_t at0 = __builtin_amdgcn_readfirstlane((many ? 16 * wave : 0) + span.first * group / step * step);
    // The next rows' queries are on their way while these are worked on.
    u32x4 next16[kSteps];
    float next_lse = 0.0f;
    auto fetch = [&](int32_t first) {
      const uint32_t at = min(first + x, rows - 1), i = group_log >= 0 ? at >> group_log : at / group, head = at - i * group;
      next_lse = lse_of[static_cast<uint64_t>(i) * static_cast<uint32_t>(c.heads) + head];
      const uint8_t* q = query + static_cast<uint64_t>(i) * static_cast<uint32_t>(2 * c.query_row_stride) +
                         static_cast<uint64_t>(head) * static_cast<uint32_t>(2 * c.query_head_stride);
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) next16[ks] = ld16_cached(q + 64 * ks);
    };
    if (at0 < end) fetch(at0);
    for (; at0 < end; at0 += step) {
      // e^(score - lse) is 2^(score * factor + less) times what the rounding of less leaves, which is 2^-11 and more for
      // logarithms of thousands.  That goes into the sums as their factor, at no instruction a score.
      const float lse = next_lse, less = lse * -a.lse_factor;
      const float past = __builtin_fmaf(lse, a.lse_rest, __builtin_fmaf(lse, a.lse_factor, less));
      const float rest = __builtin_isfinite(less) ? past : 0.0f;
      const float give = __builtin_amdgcn_exp2f(-rest);
      u32x4 rows16[kSteps];
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) rows16[ks] = next16[ks];
      fetch(at0 + step);  // behind the last ones: the last row again
      const bool gives = at0 + x < rows && lse != -__builtin_inff();
      const int32_t pos_lo = w.before + at0 / group, pos_hi = w.before + min(at0 + 15, rows - 1) / group;
      const bool plain = whole && v0 >= w.front && last <= pos_lo && (a.window == 0 || from > pos_hi - a.window) &&
                         ballot(!gives) == 0;
      uint32_t seen[4];
      if (!plain) {
        const int32_t at = min(at0 + x, rows - 1);
        const RowSight sight{w.before + at / group, nullptr};
#pragma unroll
        for (int r = 0; r < 4; ++r)
          seen[r] = (gives ? row_bits(a, w, sight, position(w, v0 + 8 * (4 * g + r))) : 0) & __shfl(unit.bits, 4 * g + r);
      }
#pragma unroll
      for (int t0 = 0; t0 < 8; t0 += kAtOnce) {
        f32x4 s[kAtOnce];
#pragma unroll
        for (int t = 0; t < kAtOnce; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks)
#pragma unroll
          for (int t = 0; t < kAtOnce; ++t) s[t] = Mma16<DT>::mma(keys[ks][t0 + t], rows16[ks], s[t]);
#pragma unroll
        for (int t = 0; t < kAtOnce; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], a.factor, less));
        if (!plain) {
#pragma unroll
          for (int t = 0; t < kAtOnce; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][r] = (seen[r] >> (t0 + t) & 1u) != 0 ? s[t][r] : 0.0f;
        }
#pragma unroll
        for (int t = 0; t < kAtOnce; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[t0 + t][r] = __builtin_fmaf(s[t][r], give, sum[t0 + t][r]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const float all = sum_of_16(sum[t][r]);
        if (x == 0) sums[wave][32 * g + 8 * r + t] = all;
      }
    __syncthreads();
    float* weights = a.weights + seq * a.weight_row_stride + kv_head * a.weight_head_stride;
    for (int32_t n = threadIdx.x; n < stride; n += WAVES * kWave) {
      const int32_t token = position(w, base + n);
      float all = many ? 0.0f : sums[n / kTilePlaces][n % kTilePlaces];
      if (many)
        for (int k = 0; k < WAVES; ++k) all += sums[k][n];
      // What no row sees, behind the end among it, gathered nothing and is not written.
      if (base + n < w.length && token < a.weight_tokens && all != 0.0f) weights[token] += all;
    }
    __syncthreads();
  }
}

template <int DT, int HD>
hipError_t launch_hd(const CacheArgs& a, dim3 grid, hipStream_t stream) {
  if constexpr (HD <= 128)
    if (a.parts == 8) {
      weights_tile_kernel<DT, HD, 8><<<grid, 8 * kWave, 0, stream>>>(a);
      return hipGetLastError();
    }
  weights_tile_kernel<DT, HD, kWavesPerBlock><<<grid, kBlockThreads, 0, stream>>>(a);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_tiles(const CacheArgs& a, dim3 grid, hipStream_t stream) {
  switch (a.r.hd) {
    case 64: return launch_hd<DT, 64>(a, grid, stream);
    case 96: return launch_hd<DT, 96>(a, grid, stream);
    case 128: return launch_hd<DT, 128>(a, grid, stream);
    case 192: return launch_hd<DT, 192>(a, grid, stream);
    default: return launch_hd<DT, 256>(a, grid, stream);
  }
}

// Whether 16 bytes of a query row can be read at a time.
bool queries_fit(const CacheAttnCall& c) {
  const int64_t most = int64_t{1} << 31;
  return ((reinterpret_cast<uint64_t>(c.query) | 2 * c.query_row_stride | 2 * c.query_head_stride) & 15) == 0 &&
         c.query_row_stride >= 0 && c.query_row_stride < most && c.query_head_stride >= 0 && c.query_head_stride < most;
}

template <int DT>
hipError_t launch(const CacheAttnCall& c, CacheArgs a, hipStream_t stream) {
  const int64_t room = c.max_blocks * c.block_size;
  int64_t longest = c.longest < room ? c.longest : room;
  if (longest > c.weight_tokens) longest = c.weight_tokens;
  const bool tiles = DT != kLinF32 && tiles_fit(c) && queries_fit(c);
  int64_t share = kBlockThreads;
  if (tiles) {
    const int64_t seq_rows = c.starts == nullptr ? 1 : (c.rows + c.batch - 1) / c.batch;
    const bool many = seq_rows * (c.heads / c.kv_heads) > 16 * (kManyTiles - 1);
    a.parts = many ? kWavesPerBlock : 1;
    share = many ? kTilePlaces : kTilePlaces * kWavesPerBlock;
  }
  int64_t groups = (longest + share - 1) / share;
  groups = groups < 1 ? 1 : groups < 4096 ? groups : 4096;
  const dim3 grid(groups, c.batch, c.kv_heads);
  // Positions for less than a workgroup per CU: eight waves share their rows (208 workgroups, 573 row tiles: 90 us,
  // with four waves 119).
  if (a.parts > 1 && groups * c.batch * c.kv_heads <= kCus) a.parts = 8;
  if constexpr (DT != kLinF32)
    if (tiles) return launch_tiles<DT>(a, grid, stream);
  weights_any_kernel<DT><<<grid, kBlockThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace
}  // namespace catt

hipError_t launch_attention_weights(const CacheAttnCall& c, hipStream_t stream) {
  const catt::CacheArgs a = catt::cache_args(c, 0);
  switch (c.dtype) {
    case kLinF32: return catt::launch<kLinF32>(c, a, stream);
    case kLinF16: return catt::launch<kLinF16>(c, a, stream);
    default: return catt::launch<kLinBF16>(c, a, stream);
  }
}

}  // namespace kvhip
