// Attention over paged caches of plain values: kv_paged_attention and kv_paged_attention_tree.
//
//   s_j = softmax_scale * sum_d q_d K[blk(j), h, d, j % bs],   lse = log sum_j e^(s_j)
//   o_d = sum_j e^(s_j - lse) V[blk(j), h, d, j % bs]
//
// over the positions j that the row sees.  One pass over the cache with a running maximum and sum in base 2; parts of a
// line (a row tile and a kv head) that run side by side leave (m, l, o) in a workspace and a second launch joins them.
#include "kv_cache_attention_tiles.h"

namespace kvhip {
namespace catt {
namespace {

// ----- any shape and type: one workgroup per (row, head, part) ------------------------------------
template <int DT>
__global__ __launch_bounds__(kBlockThreads) void cache_any_kernel(const CacheArgs a) {
  const AttnCall& c = a.r.c;
  const int64_t t = blockIdx.x, hq = blockIdx.y;
  const int32_t part = blockIdx.z;
  const int64_t line = t * c.heads + hq;
  __shared__ float q[kVisitDims];
  __shared__ VisitScratch scratch[kWavesPerBlock];
  __shared__ float acc_of[kWavesPerBlock][kVisitDims];
  __shared__ float m_of[kWavesPerBlock], l_of[kWavesPerBlock];
  const int lane = lane_id(), wave = wave_in_block();

  const RowSeq row = row_sequence(c, t);
  if (row.seq < 0) {
    if (part != 0) return;
    if (c.fill_rows)
      for (int64_t d = threadIdx.x; d < c.head_dim; d += kBlockThreads) store_o<DT>(c.out, line * c.head_dim + d, 0.0f);
    if (threadIdx.x == 0) {
      if (c.lse != nullptr) c.lse[line] = -__builtin_inff();
      if (a.parts > 1) *line_of(a, line) = Line{0, 0, 0, 0};
    }
    return;
  }
  const int32_t seq = static_cast<int32_t>(row.seq), first = static_cast<int32_t>(row.first);
  const int32_t i = static_cast<int32_t>(t) - first;
  const View w = make_view(a, seq, static_cast<int32_t>(row.count), i, i);
  const int32_t count = part_count(a, w.length);
  if (part == 0 && threadIdx.x == 0 && a.parts > 1) *line_of(a, line) = Line{count, static_cast<int32_t>(t), 1, 0};
  if (part >= count) return;
  const Span span = part_places(a, w.length, part, count);
  for (int64_t d = threadIdx.x; d < c.head_dim; d += kBlockThreads)
    q[d] = load_q<DT>(c.query, t * c.query_row_stride + hq * c.query_head_stride + d);
  __syncthreads();
  const RowSight sight = row_sight(a, w, first, i);
  const int64_t at = slot_row(a, line, part, 0);
  constexpr int kMine = kVisitDims / kBlockThreads;
  float out[kMine] = {};
  for (float lower = 0.0f;; lower = kLower) {
    float m, l, acc[kVisitDims / kWave];
    visit_row<DT, kVisitDims>(a, w, seq, sight, static_cast<int32_t>(hq) / a.r.group, q,
                              static_cast<int32_t>(span.lo) + wave * kWave, static_cast<int32_t>(span.hi), kBlockThreads,
                              lower, scratch[wave], m, l, acc);
    if (lane == 0) {
      m_of[wave] = m;
      l_of[wave] = l;
    }
#pragma unroll
    for (int i = 0; i < kVisitDims / kWave; ++i)
      if (lane + i * kWave < c.head_dim) acc_of[wave][lane + i * kWave] = acc[i];
    __syncthreads();
    float top = m_of[0];
    for (int x = 1; x < kWavesPerBlock; ++x) top = fmaxf(top, m_of[x]);
    float fade[kWavesPerBlock], sum = 0.0f;
    for (int x = 0; x < kWavesPerBlock; ++x) {
      fade[x] = fade_to(m_of[x], top);
      sum += l_of[x] * fade[x];
    }
    bool over = false;
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int64_t d = threadIdx.x + k * kBlockThreads;
      if (d >= c.head_dim) break;
      float o = 0.0f;
      for (int x = 0; x < kWavesPerBlock; ++x) o += acc_of[x][d] * fade[x];
      if (lower == 0.0f || !__builtin_isfinite(out[k])) out[k] = sum == 0.0f ? 0.0f : o / sum;
      over |= !__builtin_isfinite(out[k]);
    }
    if (lower == 0.0f && threadIdx.x == 0) {
      if (count > 1) {
        slot_ml(a, at)[0] = top;
        slot_ml(a, at)[1] = sum;
      } else if (c.lse != nullptr) {
        c.lse[line] = log_sum(top, sum);
      }
    }
    if (DT == kLinF16 || lower != 0.0f || !__builtin_isfinite(sum)) break;
    if (__syncthreads_or(over) == 0) break;
  }
#pragma unroll
  for (int k = 0; k < kMine; ++k) {
    const int64_t d = threadIdx.x + k * kBlockThreads;
    if (d >= c.head_dim) break;
    if (count > 1) slot_out(a, at)[d] = out[k];
    else store_o<DT>(c.out, line * c.head_dim + d, out[k]);
  }
}

// ----- join -----------------------------------------------------------------------------------------
// The mean of the parts' outputs, weighted by their sums.  One workgroup per row of a line.  Its waves take the parts in
// turn, in the same order in every run.
template <int DT>
__global__ __launch_bounds__(kBlockThreads) void cache_join_kernel(const CacheArgs a) {
  const AttnCall& c = a.r.c;
  const int64_t line = blockIdx.x;
  const int32_t x = blockIdx.y;
  const Line info = *line_of(a, line);
  if (info.parts <= 1) return;
  // The form for any shape has a line per (row, head); the tiles' rows are (position, head of the group).
  int64_t row, head;
  if (a.tiles == 0) {
    row = info.first;
    head = line - row * c.heads;
  } else {
    const int32_t at = info.base + x;
    if (at >= info.count * a.r.group) return;
    row = info.first + at / a.r.group;
    head = (line % c.kv_heads) * a.r.group + at % a.r.group;
  }
  __shared__ float acc_of[kWavesPerBlock][kVisitDims];
  __shared__ float top_of[kWavesPerBlock], sum_of[kWavesPerBlock];
  const int lane = lane_id(), wave = wave_in_block();
  const float* ml = slot_ml(a, slot_row(a, line, 0, x));
  const int64_t pitch = 2 * static_cast<int64_t>(a.slot_rows);
  float top = -__builtin_inff();
  for (int32_t s = threadIdx.x; s < info.parts; s += kBlockThreads) top = fmaxf(top, ml[s * pitch]);
  top = wave_max(top);
  if (lane == 0) top_of[wave] = top;
  __syncthreads();
  for (int k = 0; k < kWavesPerBlock; ++k) top = fmaxf(top, top_of[k]);
  float acc[kVisitDims / kWave] = {}, sum = 0.0f;
  for (int32_t s = threadIdx.x; s < info.parts; s += kBlockThreads) sum += ml[s * pitch + 1] * fade_to(ml[s * pitch], top);
  sum = wave_sum(sum);
  if (lane == 0) sum_of[wave] = sum;
  __syncthreads();
  sum = 0.0f;
  for (int k = 0; k < kWavesPerBlock; ++k) sum += sum_of[k];
  const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
  const float* part = slot_out(a, slot_row(a, line, 0, x));
  const int64_t step = static_cast<int64_t>(a.slot_rows) * c.head_dim;
#pragma unroll 4
  for (int32_t s = wave; s < info.parts; s += kWavesPerBlock) {
    const float share = ml[s * pitch + 1] * fade_to(ml[s * pitch], top) * scale;
#pragma unroll
    for (int i = 0; i < kVisitDims / kWave; ++i)
      if (lane + i * kWave < c.head_dim) acc[i] = __builtin_fmaf(part[s * step + lane + i * kWave], share, acc[i]);
  }
#pragma unroll
  for (int i = 0; i < kVisitDims / kWave; ++i)
    if (lane + i * kWave < c.head_dim) acc_of[wave][lane + i * kWave] = acc[i];
  __syncthreads();
  const int64_t out = row * c.heads + head;
  for (int64_t d = threadIdx.x; d < c.head_dim; d += kBlockThreads) {
    float o = 0.0f;
    for (int k = 0; k < kWavesPerBlock; ++k) o += acc_of[k][d];
    store_o<DT>(c.out, out * c.head_dim + d, o);
  }
  if (threadIdx.x == 0 && c.lse != nullptr) c.lse[out] = log_sum(top, sum);
}

// The same with a wave per row, for few parts (the rows of 16 trees in three parts: 14 us, with a workgroup each 36).
template <int DT>
__global__ __launch_bounds__(kBlockThreads) void cache_join_few_kernel(const CacheArgs a) {
  const AttnCall& c = a.r.c;
  const int64_t line = blockIdx.x;
  const int32_t x = blockIdx.y * kWavesPerBlock + wave_in_block();
  const Line info = *line_of(a, line);
  const int32_t at = info.base + x;
  if (info.parts <= 1 || x >= a.slot_rows || at >= info.count * a.r.group) return;
  const int64_t row = info.first + at / a.r.group, head = (line % c.kv_heads) * a.r.group + at % a.r.group;
  const int lane = lane_id();
  const float* ml = slot_ml(a, slot_row(a, line, 0, x));
  const float* part = slot_out(a, slot_row(a, line, 0, x));
  const int64_t pitch = 2 * static_cast<int64_t>(a.slot_rows), step = static_cast<int64_t>(a.slot_rows) * c.head_dim;
  float top = -__builtin_inff(), sum = 0.0f;
  for (int32_t s = 0; s < info.parts; ++s) top = fmaxf(top, ml[s * pitch]);
  for (int32_t s = 0; s < info.parts; ++s) sum += ml[s * pitch + 1] * fade_to(ml[s * pitch], top);
  const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
  constexpr int kDims = 256 / kWave;  // of the forms in tiles
  float acc[kDims] = {};
  for (int32_t s = 0; s < info.parts; ++s) {
    const float share = ml[s * pitch + 1] * fade_to(ml[s * pitch], top) * scale;
#pragma unroll
    for (int i = 0; i < kDims; ++i)
      if (lane + i * kWave < c.head_dim) acc[i] = __builtin_fmaf(part[s * step + lane + i * kWave], share, acc[i]);
  }
  const int64_t out = row * c.heads + head;
#pragma unroll
  for (int i = 0; i < kDims; ++i)
    if (lane + i * kWave < c.head_dim)
      store_o<DT>(c.out, out * c.head_dim + lane + i * kWave, acc[i]);
  if (lane == 0 && c.lse != nullptr) c.lse[out] = log_sum(top, sum);
}

// The most places that a line's view has, by `longest` and what a table row has room for.
int64_t most_places(const CacheAttnCall& c, int rows) {
  const int64_t room = c.max_blocks * c.block_size;
  int64_t longest = c.longest < room ? c.longest : room;
  if (longest < 1) longest = 1;
  if (c.window <= 0) return longest;
  // A window of each of a tile's positions, the first tokens, and both rounded to 16.
  const int64_t group = c.heads / c.kv_heads;
  const int64_t positions = c.starts == nullptr ? 1 : (rows + group - 1) / group + 1;
  const int64_t sinks = c.sinks < room ? c.sinks : room, window = c.window < room ? c.window : room;
  const int64_t reach = window + positions - 1 + 15 + (sinks + 15) / 16 * 16;
  return reach < longest ? reach : longest;
}

// The form for any shape, which is there to be right: parts of 1024 positions or more.
constexpr int64_t kAnyPart = 1024;
constexpr int64_t kAnyParts = 64;
constexpr int64_t kAnyGroups = 8192;  // workgroups from which on a line is not cut further

// How a call is cut.  size: rows of a tile (0: the form for any shape).
struct Plan {
  int64_t size, lines, parts, part, slot_rows, tiles;
};

// Few rows: parts of whole turns of a workgroup, as many as make kRowsGroups workgroups (48 decode rows of 295 to 8192
// tokens, us: 768 193, 1600 180, 2048 178 to 188, 4096 182, 8192 187; 16 rows of 2048 visible ones 55, then 48).
constexpr int64_t kTurnPlaces = kTilePlaces * kWavesPerBlock;
constexpr int64_t kRowsGroups = 2048;
constexpr int64_t kFewRows = 32;
constexpr int64_t kAtOnce = 512;  // two workgroups a CU
// Many rows (16 trees of 34 to 64 tokens over 620 to 4001, us: 320 157, 640 124, 1024 103, 1536 126, 2048 131; two chunks
// of 1753 and 2048 rows, whose tiles alone make 960: uncut 432, in two parts 504).
constexpr int64_t kWidePlaces = 512;
constexpr int64_t kWideGroups = 1024;

// Parts of a multiple of `unit` places each: no more than give `groups` workgroups, and `most` of a line.
void cut(Plan& p, int64_t places, int64_t unit, int64_t groups, int64_t most) {
  int64_t parts = groups / (p.lines > 0 ? p.lines : 1);
  parts = parts < 1 ? 1 : parts < most ? parts : most;
  p.part = ((places + parts - 1) / parts + unit - 1) / unit * unit;
  p.parts = (places + p.part - 1) / p.part;
}

// Whether the scaling of scores may be fused with the difference to their maximum, as the form for many rows does it: the
// factor is positive, and -inf times it is -inf.
bool fuses_scale(const CacheAttnCall& c) { return c.softmax_scale > 1e-30 && c.softmax_scale < 1e30; }

Plan make_plan(const CacheAttnCall& c) {
  Plan p{};
  if (tiles_fit(c)) {
    const int64_t group = c.heads / c.kv_heads;
    const int64_t seq_rows = (c.starts == nullptr || c.batch == 0 ? 1 : (c.rows + c.batch - 1) / c.batch) * group;
    // Few rows, and calls so small that all of their tiles of 16 rows run at once: those take the shortest way through a
    // line (three trees of 7 to 13 tokens over 400: 12 us, in wide tiles 28).
    const int64_t turns = (most_places(c, 16) + kTurnPlaces - 1) / kTurnPlaces;
    const bool all_at_once = (c.rows * group / 16 + c.batch) * c.kv_heads * turns <= kAtOnce;
    const bool wide = seq_rows > kFewRows && c.head_dim <= 128 && fuses_scale(c) && !all_at_once;
    p.size = wide ? kWideTileRows : seq_rows <= 16 || c.head_dim > 128 || all_at_once ? 16 : 32;
    CacheArgs a = cache_args(c, static_cast<int>(p.size));
    p.tiles = tiles_bound(a.r.c, static_cast<int>(p.size));
    if (p.tiles < 1) p.tiles = 1;  // rows of no sequence
    p.lines = p.tiles * c.kv_heads;
    p.slot_rows = c.starts == nullptr && group < p.size ? group : p.size;
    const int64_t places = most_places(c, static_cast<int>(p.size));
    if (wide) cut(p, places, kWidePlaces, kWideGroups, 64);
    else cut(p, places, kTurnPlaces, kRowsGroups, 256);
    return p;
  }
  p.lines = c.rows * c.heads;
  p.slot_rows = 1;
  cut(p, most_places(c, 1), kAnyPart, kAnyGroups, kAnyParts);
  return p;
}

int64_t plan_workspace(const CacheAttnCall& c, const Plan& p) {
  if (p.parts <= 1) return 0;
  const int64_t slots = p.lines * p.parts * p.slot_rows;
  return (ml_floats(slots) + slots * c.head_dim) * 4 + p.lines * static_cast<int64_t>(sizeof(Line));
}

constexpr int64_t kFewParts = 8;

template <int DT>
hipError_t launch(const CacheAttnCall& c, const Plan& p, CacheArgs a, hipStream_t stream) {
  hipError_t err;
  if (p.size > 0) {
    err = p.size == kWideTileRows ? launch_wide_tiles(a, stream) : launch_rows(a, static_cast<int>(p.size / 16), stream);
  } else {
    cache_any_kernel<DT><<<dim3(c.rows, c.heads, p.parts), kBlockThreads, 0, stream>>>(a);
    err = hipGetLastError();
  }
  if (err != hipSuccess) return err;
  if (p.parts > 1) {
    if (p.size > 0 && p.parts <= kFewParts)
      cache_join_few_kernel<DT><<<dim3(p.lines, (p.slot_rows + kWavesPerBlock - 1) / kWavesPerBlock), kBlockThreads, 0, stream>>>(a);
    else
      cache_join_kernel<DT><<<dim3(p.lines, p.slot_rows), kBlockThreads, 0, stream>>>(a);
  }
  return hipGetLastError();
}

}  // namespace

bool tiles_fit(const CacheAttnCall& c) {
  if (c.dtype != kLinF16 && c.dtype != kLinBF16) return false;
  const int64_t hd = c.head_dim;
  if (c.block_size % 8 != 0 || (hd != 64 && hd != 96 && hd != 128 && hd != 192 && hd != 256)) return false;
  if ((reinterpret_cast<uint64_t>(c.out) & 7) != 0 || c.kv_heads > 65535) return false;
  for (int kv = 0; kv < 2; ++kv)
    if (c.cache[kv] != nullptr && (((reinterpret_cast<uint64_t>(c.cache[kv]) | c.cache_block_stride[kv]) & 15) != 0 ||
                                   c.cache_block_stride[kv] < 0 || c.cache_block_stride[kv] >= int64_t{1} << 32))
      return false;
  return true;
}

CacheArgs cache_args(const CacheAttnCall& c, int size) {
  AttnCall k{};
  k.query = c.query;
  k.out = c.out;
  k.lse = c.lse;
  for (int kv = 0; kv < 2; ++kv) {
    k.cache[kv] = c.cache[kv];
    k.cache_block_stride[kv] = c.cache_block_stride[kv];
  }
  k.tables = c.tables;
  k.lens = c.lens;
  k.starts = c.starts;
  k.workspace = c.workspace;
  k.rows = c.rows;
  k.batch = c.batch;
  k.heads = c.heads;
  k.kv_heads = c.kv_heads;
  k.head_dim = c.head_dim;
  k.block_size = c.block_size;
  k.num_blocks = c.num_blocks;
  k.max_blocks = c.max_blocks;
  k.query_row_stride = c.query_row_stride;
  k.query_head_stride = c.query_head_stride;
  k.table_stride = c.table_stride;
  k.softmax_scale = c.softmax_scale;
  k.dtype = c.dtype;
  k.wide_tables = c.wide_tables;
  k.wide_lens = c.wide_lens;
  k.wide_starts = c.wide_starts;
  k.fill_rows = c.fill_rows;
  CacheArgs a{};
  a.r.c = k;
  a.r.batch = static_cast<int32_t>(c.batch);
  a.r.heads = static_cast<int32_t>(c.heads);
  a.r.hd = static_cast<int32_t>(c.head_dim);
  a.r.bs = static_cast<int32_t>(c.block_size);
  a.r.num_blocks = static_cast<int32_t>(c.num_blocks);
  a.r.room = static_cast<int32_t>(c.max_blocks * c.block_size);
  a.r.group = static_cast<int32_t>(c.heads / c.kv_heads);
  a.r.block_shift = (c.block_size & (c.block_size - 1)) == 0 ? __builtin_ctzll(c.block_size) : -1;
  a.r.seq_tiles = size > 0 ? (a.r.group + size - 1) / size : 1;
  a.masks = c.masks;
  a.mask_stride = c.mask_stride;
  a.mask_words = static_cast<int32_t>(c.mask_words);
  a.weights = c.weights;
  a.weight_row_stride = c.weight_row_stride;
  a.weight_head_stride = c.weight_head_stride;
  a.weight_tokens = static_cast<int32_t>(c.weight_tokens < kMostRoom ? c.weight_tokens : kMostRoom);
  a.window = static_cast<int32_t>(c.window < kMostRoom ? c.window : kMostRoom);
  a.sinks = static_cast<int32_t>(c.sinks < kMostRoom ? c.sinks : kMostRoom);
  a.scale = static_cast<float>(c.softmax_scale);
  a.factor = static_cast<float>(c.softmax_scale * 1.4426950408889634);
  const bool ratio = a.factor != 0.0f && __builtin_isfinite(a.factor);
  const double per_lse = ratio ? a.factor / c.softmax_scale : 1.4426950408889634;
  a.lse_factor = static_cast<float>(per_lse);
  a.lse_rest = static_cast<float>(per_lse - a.lse_factor);
  a.scale_rest = __builtin_isfinite(a.scale) ? static_cast<float>(c.softmax_scale - a.scale) : 0.0f;
  return a;
}

}  // namespace catt

int64_t cache_attention_workspace(const CacheAttnCall& c) { return catt::plan_workspace(c, catt::make_plan(c)); }

hipError_t launch_cache_attention(const CacheAttnCall& c, hipStream_t stream) {
  const catt::Plan p = catt::make_plan(c);
  catt::CacheArgs a = catt::cache_args(c, static_cast<int>(p.size));
  a.part = static_cast<int32_t>(p.part);
  a.parts = static_cast<int32_t>(p.parts);
  a.slot_rows = static_cast<int32_t>(p.slot_rows);
  a.tiles = static_cast<int32_t>(p.tiles);
  a.lines = p.lines;
  switch (c.dtype) {
    case kLinF32: return catt::launch<kLinF32>(c, p, a, stream);
    case kLinF16: return catt::launch<kLinF16>(c, p, a, stream);
    default: return catt::launch<kLinBF16>(c, p, a, stream);
  }
}

}  // namespace kvhip
