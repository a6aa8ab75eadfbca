// FP8 store into paged caches with one scale per (block, head): kv_linear_to_paged_fp8_block.
//
// Per layer, block b, kv head h and plane, with N the finite new values of the block and F the format's
// largest value (448 / 57344):
//   anew = column 0 is written, or the old scale is not positive and finite
//   s    = max(max|N| / F, 2^-60, anew ? 0 : s_old)
//   written column: encode(x / s);  other columns: 0 if anew, as they are if s == s_old, else
//   encode(decode(code) * s_old / s)
// all in fp32 with one rounding per operation, so the result does not depend on how the work is cut.
//
// The tokens of a block may stand anywhere in the call.  A block's leader, the token that owns its lowest written
// column, names the block once; which token writes a column comes from the claim tags of the call or, for up to
// kStoreScanTokens tokens, from the slots themselves, which every workgroup reads (one launch, no tags).
//
// A unit is one (block, plane, head, layer), done by one wave.  Where rows and blocks allow it (16-token groups
// of columns, 8-dim pieces, 16-byte addresses) the wave loads 16-byte pieces of 4 tokens at a time, lane (tg, pc)
// the tokens of columns 4 tg .. 4 tg + 3 and dims 8 pc .. 8 pc + 7, so that four codes of a dim are one dword of
// the cache; two exchanges between the four lanes of a piece (v_permlane32_swap, v_permlane16_swap) then give
// every lane whole 16-column rows of two dims.  Other shapes go element by element.
// What bounds it: few tokens, latency (a token's row, its block's scale, the stores); many, memory and the ten or so
// operations that a value takes (E4M3, whose small quotients are more often there to be flushed, is the slower).
// Measured: 64 tokens of 8 x 128 bf16 into pages of 16, 5.2 us; 30977 tokens, 52 us with the check of the slots
// (3.7 TB/s; a large copy 4.7); 16 layers of 4001 tokens fp16 into pages of 64, 116 us (179 with the pieces read
// twice), of bf16 as E4M3 135 us.
#include "kv_serving.h"

namespace kvhip {
namespace {

template <int CODEC>
constexpr float kCodecMax = CODEC == kE4M3 ? 448.0f : 57344.0f;

struct StoreArgs {
  BlockStoreParams p;
  int32_t window;  // tokens per workgroup (claims form)
};

template <int LDT>
__device__ __forceinline__ float load_lin(const void* base, int64_t i) {
  if constexpr (LDT == kLinF32) return static_cast<const float*>(base)[i];
  else return lin_to_f32<LDT>(static_cast<const uint16_t*>(base)[i]);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// Which token writes a column of the block, or -1.
struct TagColumns {
  const uint64_t* tags;  // of the block's first column
  uint32_t epoch;
  __device__ __forceinline__ int32_t operator()(int64_t col) const {
    const uint64_t tag = tags[col];
    return static_cast<uint32_t>(tag >> 32) == epoch ? static_cast<int32_t>(tag & 0xFFFFFFFFu) - 1 : -1;
  }
};
struct MapColumns {
  const int32_t* map;  // LDS, token + 1 or 0
  __device__ __forceinline__ int32_t operator()(int64_t col) const { return map[col] - 1; }
};

struct Unit {
  const uint8_t* lin;  // the head's first element of token 0
  int64_t token_bytes;
  uint8_t* codes;      // [head_dim][block_size]
  float* scale;
  int64_t hd, bs;
};

__device__ __forceinline__ Unit unit_of(const BlockStoreParams& p, int elt, int64_t block, int64_t layer, int64_t head,
                                        int kv) {
  Unit u;
  u.lin = static_cast<const uint8_t*>(p.lin[kv]) + (layer * p.lin_layer_stride + head * p.head_dim) * elt;
  u.token_bytes = p.lin_token_stride * elt;
  u.codes = p.cache[kv] + layer * p.layer_stride[kv] + block * p.block_stride[kv] + head * p.head_dim * p.block_size;
  u.scale = p.scale[kv] + (layer * p.num_blocks + block) * p.num_heads + head;
  u.hd = p.head_dim;
  u.bs = p.block_size;
  return u;
}

template <int CODEC>
__device__ __forceinline__ float new_scale(float most, float before, bool anew) {
  const float now = fmaxf(div_rn(most, kCodecMax<CODEC>), kScaleFloor);
  return anew ? now : fmaxf(now, before);
}

// ----- element by element -----------------------------------------------------------------------
template <int CODEC, int LDT, typename COLUMNS>
__device__ __forceinline__ void store_unit(const Unit& u, const COLUMNS& token_of) {
  constexpr int kElt = LDT == kLinF32 ? 4 : 2;
  float most = 0.0f;
  for (int64_t col = 0; col < u.bs; ++col) {
    const int64_t tok = token_of(col);
    if (tok < 0) continue;
    for (int64_t d = lane_id(); d < u.hd; d += kWave) {
      const float x = fabsf(load_lin<LDT>(u.lin + tok * u.token_bytes, d));
      most = fmaxf(most, x < __builtin_inff() ? x : 0.0f);
    }
  }
  most = wave_max(most);
  const float before = *u.scale;
  const bool anew = token_of(0) >= 0 || scale_refused(before);
  const float now = new_scale<CODEC>(most, before, anew);
  for (int64_t col = 0; col < u.bs; ++col) {
    const int64_t tok = token_of(col);
    if (tok < 0 && !anew && now == before) continue;
    for (int64_t d = lane_id(); d < u.hd; d += kWave) {
      uint8_t* at = u.codes + d * u.bs + col;
      uint32_t code = 0;
      if (tok >= 0) code = fp8_encode<CODEC>(div_rn(load_lin<LDT>(u.lin + tok * u.token_bytes, d), now));
      else if (!anew) code = fp8_encode<CODEC>(div_rn(fp8_decode<CODEC>(*at) * before, now));
      *at = static_cast<uint8_t>(code);
    }
  }
  static_assert(kElt == 4 || kElt == 2, "");
  if (lane_id() == 0) *u.scale = now;
}

// ----- by 16-byte pieces ------------------------------------------------------------------------
template <int LDT>
struct Piece {  // 8 dims of a token
  u32x4 raw[LDT == kLinF32 ? 2 : 1];
  __device__ __forceinline__ float at(int j) const {
    if constexpr (LDT == kLinF32) return __uint_as_float(raw[j >> 2][j & 3]);
    else return lin_to_f32<LDT>(elem16(raw[0], j));
  }
};

// The pieces of dims 128 `chunk` + 8 pc .. + 7 of the lane's four columns of group `group`; absent tokens are 0.
template <int LDT>
__device__ __forceinline__ void load_pieces(const Unit& u, const int32_t* tok, int chunk, Piece<LDT>* x) {
  const int64_t d = 128 * chunk + 8 * (lane_id() & 15);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = Piece<LDT>{};
    if (tok[i] >= 0 && d < u.hd) {
      const uint8_t* p = u.lin + tok[i] * u.token_bytes + d * (LDT == kLinF32 ? 4 : 2);
      x[i].raw[0] = ld16_cached(p);
      if constexpr (LDT == kLinF32) x[i].raw[1] = ld16_cached(p + 16);
    }
  }
}

// Tokens of the lane's four columns of a group; returns which of its 16 columns are written.
template <typename COLUMNS>
__device__ __forceinline__ uint32_t group_tokens(const COLUMNS& token_of, int64_t group, int32_t* tok) {
  const int32_t mine = token_of(16 * group + (lane_id() & 15));
#pragma unroll
  for (int i = 0; i < 4; ++i) tok[i] = __shfl(mine, 4 * (lane_id() >> 4) + i);
  return static_cast<uint32_t>(ballot(mine >= 0)) & 0xFFFFu;
}

template <int LDT>
__device__ __forceinline__ float most_of(const Piece<LDT>* x, float most) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = fabsf(x[i].at(j));
      most = fmaxf(most, v < __builtin_inff() ? v : 0.0f);
    }
  return most;
}

// The largest magnitude bits of the pieces, for 16-bit values those of two in the halves of a dword: one or two
// operations a value, where values with their infinities and NaN left out (most_of) take five.
template <int LDT>
__device__ __forceinline__ uint32_t top_bits(const Piece<LDT>* x, uint32_t top) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int w = 0; w < (LDT == kLinF32 ? 8 : 4); ++w) {
      if constexpr (LDT == kLinF32)
        top = max(top, x[i].raw[w >> 2][w & 3] & 0x7FFFFFFFu);
      else
        top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                                                     __builtin_bit_cast(u16x2, x[i].raw[0][w] & 0x7FFF7FFFu)));
    }
  return top;
}

// The magnitude behind a lane's top_bits; with infinities and NaN at or past kInfinity.
template <int LDT>
constexpr uint32_t kInfinity = LDT == kLinF32 ? 0x7F800000u : LDT == kLinF16 ? 0x7C00u : 0x7F80u;

template <int LDT>
__device__ __forceinline__ uint32_t wave_top(uint32_t top) {
  if constexpr (LDT != kLinF32) top = max(top & 0xFFFFu, top >> 16);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o)));
  return __builtin_amdgcn_readfirstlane(top);
}

template <int LDT>
__device__ __forceinline__ float top_value(uint32_t bits) {
  if constexpr (LDT == kLinF32) return __uint_as_float(bits);
  else return lin_to_f32<LDT>(static_cast<uint16_t>(bits));
}

// Bytes of columns 4 k .. 4 k + 3 that are written, as a mask of the dword.
__device__ __forceinline__ uint32_t column_bytes(uint32_t written, int k) {
  return (((written >> (4 * k) & 15u) * 0x00204081u) & 0x01010101u) * 0xFFu;
}

// The four lanes of a piece trade their dwords: in, dword j holds dim j of the lane's columns; out, row r holds
// the 16 columns of dim 2 tg + r.
__device__ __forceinline__ void trade(uint32_t* w, u32x4* row) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const auto s = __builtin_amdgcn_permlane32_swap(w[j], w[j + 4], false, false);
    w[j] = s[0];
    w[j + 4] = s[1];
  }
#pragma unroll
  for (int j = 0; j < 8; j += 4)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const auto s = __builtin_amdgcn_permlane16_swap(w[j + r], w[j + 2 + r], false, false);
      row[r][j / 2] = s[0];
      row[r][j / 2 + 1] = s[1];
    }
}

template <int CODEC>
__device__ __forceinline__ uint32_t recode(uint32_t w, float before, float now) {
  uint32_t out = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    out |= fp8_encode<CODEC>(div_rn(fp8_decode<CODEC>(w >> (8 * k) & 0xFFu) * before, now)) << (8 * k);
  return out;
}

// HELD > 0: the block is HELD groups of at most 128 dims, whose pieces stay in registers between the two passes; else
// the second pass reads them again (from memory: what the chip's waves read between the two is more than its L2).
template <int CODEC, int LDT, int HELD, typename COLUMNS>
__device__ __forceinline__ void store_unit_pieces(const Unit& u, const COLUMNS& token_of) {
  constexpr int kHeld = HELD > 0 ? HELD : 1;
  const int groups = HELD > 0 ? HELD : static_cast<int>(u.bs >> 4);
  const int chunks = HELD > 0 ? 1 : static_cast<int>((u.hd + 127) >> 7);
  const float before = *u.scale;
  int32_t tok[kHeld][4];
  uint32_t mask[kHeld], top = 0;
  Piece<LDT> pieces[kHeld][4];
  // The groups' pieces one after the other, or all that are held.
  auto each_group = [&](auto&& see) {
    if constexpr (HELD > 0) {
#pragma unroll
      for (int g = 0; g < HELD; ++g) see(pieces[g]);
    } else {
      for (int g = 0; g < groups; ++g) {
        if (group_tokens(token_of, g, tok[0]) == 0) continue;
        for (int ch = 0; ch < chunks; ++ch) {
          load_pieces<LDT>(u, tok[0], ch, pieces[0]);
          see(pieces[0]);
        }
      }
    }
  };
  if constexpr (HELD > 0) {  // all on their way together
#pragma unroll
    for (int g = 0; g < HELD; ++g) mask[g] = group_tokens(token_of, g, tok[g]);
#pragma unroll
    for (int g = 0; g < HELD; ++g) load_pieces<LDT>(u, tok[g], 0, pieces[g]);
  }
  each_group([&](const Piece<LDT>* x) { top = top_bits<LDT>(x, top); });
  top = wave_top<LDT>(top);
  const bool odd = top >= kInfinity<LDT>;
  float most = 0.0f;
  if (odd) {
    each_group([&](const Piece<LDT>* x) { most = most_of<LDT>(x, most); });
    most = wave_max(most);
  } else {
    most = top_value<LDT>(top);
  }
  const bool anew = token_of(0) >= 0 || scale_refused(before);
  const float now = new_scale<CODEC>(most, before, anew);
  const bool same = !anew && now == before;
  // The quotient with one hoisted reciprocal is exact for scales in [2^-60, 2^60) and every finite value: a value
  // so small that its residuals underflow has a quotient below 2^-40, which is flushed either way.
  const bool exact = !odd && now < 0x1p60f;
  const float r = div_rn(1.0f, now);
  const int tg = lane_id() >> 4, pc = lane_id() & 15;
#pragma unroll kHeld
  for (int g = 0; g < groups; ++g) {
    const uint32_t written = HELD > 0 ? mask[HELD > 0 ? g : 0] : group_tokens(token_of, g, tok[0]);
    Piece<LDT>* x = pieces[HELD > 0 ? g : 0];
    if (written == 0 && same) continue;
    for (int ch = 0; ch < chunks; ++ch) {
      if (HELD == 0) load_pieces<LDT>(u, tok[0], ch, x);
      uint32_t w[8];
      u32x4 row[2];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (exact) {
          constexpr bool kNarrow = LDT != kLinF32;
          w[j] = fp8_pack4_hw<CODEC>(quot_fast<kNarrow>(x[0].at(j), now, r), quot_fast<kNarrow>(x[1].at(j), now, r),
                                     quot_fast<kNarrow>(x[2].at(j), now, r), quot_fast<kNarrow>(x[3].at(j), now, r));
        } else {
          w[j] = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[j] |= fp8_encode<CODEC>(div_rn(x[i].at(j), now)) << (8 * i);
        }
      }
      trade(w, row);
      const int64_t d = 128 * ch + 8 * pc + 2 * tg;
      if (d >= u.hd) continue;
      uint8_t* at = u.codes + d * u.bs + 16 * g;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (written != 0xFFFFu) {
          u32x4 old = {0, 0, 0, 0};
          if (!anew) old = ld16_cached(at + k * u.bs);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t m = column_bytes(written, q);
            if (!anew && !same) old[q] = recode<CODEC>(old[q], before, now);
            row[k][q] = (row[k][q] & m) | (old[q] & ~m);
          }
        }
        st16_cached(at + k * u.bs, row[k]);
      }
    }
  }
  if (lane_id() == 0) *u.scale = now;
}

// By elements, by pieces, or by pieces of which a block's kHeldPieces + n - 1 groups are held.
enum StoreForm : int { kElements = 0, kPieces = 1, kHeldPieces = 2, kHeldPieces2 = 3, kHeldPieces4 = 5 };

template <int CODEC, int LDT, int FORM, typename COLUMNS>
__device__ __forceinline__ void store_one(const BlockStoreParams& p, int64_t block, int64_t layer, int64_t unit,
                                          const COLUMNS& token_of) {
  const Unit u = unit_of(p, LDT == kLinF32 ? 4 : 2, block, layer, unit >> 1, static_cast<int>(unit & 1));
  if constexpr (FORM == kElements) store_unit<CODEC, LDT>(u, token_of);
  else store_unit_pieces<CODEC, LDT, FORM - kPieces>(u, token_of);
}

// Few tokens: one workgroup per (token, four units, layer), which makes its block's columns from all the slots.
template <int CODEC, int LDT, int FORM>
__global__ __launch_bounds__(kBlockThreads) void block_store_scan_kernel(const StoreArgs a) {
  const BlockStoreParams& p = a.p;
  __shared__ int32_t map[kStoreScanColumns];
  __shared__ int refused, lowest;
  const int64_t bs = p.block_size, slots_all = p.num_blocks * bs;
  const int64_t slot = p.slots[blockIdx.x];
  const int64_t block = slot < 0 ? -1 : slot / bs;
  const int64_t mine = threadIdx.x < p.num_tokens ? p.slots[threadIdx.x] : -1;
  if (threadIdx.x == 0) {
    refused = 0;
    lowest = kStoreScanColumns;
  }
  for (int c = threadIdx.x; c < bs; c += kBlockThreads) map[c] = 0;
  __syncthreads();
  if (mine >= slots_all) refused = 1;
  if (block >= 0 && mine >= block * bs && mine < (block + 1) * bs) {
    const int col = static_cast<int>(mine - block * bs);
    atomicMax(&map[col], static_cast<int>(threadIdx.x) + 1);
    atomicMin(&lowest, col);
  }
  __syncthreads();
  if (p.check.report != nullptr) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0)
      __hip_atomic_store(p.check.report, 2 * p.check.stamp + refused, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    if (refused) return;
  }
  if (block < 0 || slot >= slots_all) return;
  if (slot - block * bs != lowest || map[lowest] != static_cast<int>(blockIdx.x) + 1) return;
  const int64_t unit = static_cast<int64_t>(blockIdx.y) * kWavesPerBlock + wave_in_block();
  if (unit < 2 * p.num_heads) store_one<CODEC, LDT, FORM>(p, block, blockIdx.z, unit, MapColumns{map});
}

// Many tokens: one workgroup per (window of tokens, share of the units, layer).
constexpr int kMostWindow = 64;

template <int CODEC, int LDT, int FORM>
__global__ __launch_bounds__(kBlockThreads) void block_store_tags_kernel(const StoreArgs a) {
  const BlockStoreParams& p = a.p;
  __shared__ int64_t leads[kMostWindow];
  __shared__ int count;
  if (refused_ahead(p.check)) return;
  const int64_t bs = p.block_size;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * a.window + threadIdx.x;
  if (static_cast<int>(threadIdx.x) < a.window && t < p.num_tokens) {
    const int64_t slot = p.slots[t];
    if (slot >= 0 && slot < p.num_blocks * bs) {
      const int64_t block = slot / bs, col = slot - block * bs;
      const TagColumns token_of{p.owner + block * bs, p.epoch};
      bool lead = true;
      for (int64_t c = 0; c < col && lead; ++c) lead = token_of(c) < 0;
      if (lead && token_of(col) == t) leads[atomicAdd(&count, 1)] = block;
    }
  }
  __syncthreads();
  // The units of this workgroup's share of every block it leads, a wave each.
  const int64_t share = (2 * p.num_heads + gridDim.y - 1) / gridDim.y;
  const int64_t first = blockIdx.y * share;
  const int64_t units = first + share < 2 * p.num_heads ? share : 2 * p.num_heads - first;
  if (units <= 0) return;
  for (int64_t i = wave_in_block(); i < count * units; i += kWavesPerBlock) {
    const int64_t b = i / units, block = uniform64(leads[b]);
    store_one<CODEC, LDT, FORM>(p, block, blockIdx.z, first + (i - b * units), TagColumns{p.owner + block * bs, p.epoch});
  }
}

__global__ __launch_bounds__(kBlockThreads) void block_tag_reset_kernel(const int64_t* slots, int64_t n,
                                                                        int64_t num_blocks, int64_t bs,
                                                                        uint64_t* owner) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlockThreads + threadIdx.x;
  const int64_t t = i / bs;
  if (t >= n) return;
  const int64_t s = slots[t];
  if (s < 0 || s >= num_blocks * bs) return;
  owner[s / bs * bs + (i - t * bs)] = 0;
}

template <int CODEC, int LDT, int FORM>
hipError_t launch_form(const BlockStoreParams& p, hipStream_t stream) {
  StoreArgs a{p, 0};
  const uint32_t layers = static_cast<uint32_t>(p.num_layers);
  if (p.owner == nullptr) {
    const dim3 grid(static_cast<uint32_t>(p.num_tokens),
                    static_cast<uint32_t>((2 * p.num_heads + kWavesPerBlock - 1) / kWavesPerBlock), layers);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(block_store_scan_kernel<CODEC, LDT, FORM>), grid, dim3(kBlockThreads), 0,
                       stream, a);
    return hipGetLastError();
  }
  // Windows as wide as leaves the chip enough workgroups: the tokens of a window may each lead a block.
  a.window = kMostWindow;
  while (a.window > kWavesPerBlock && p.num_tokens < int64_t{128} * a.window) a.window /= 2;
  const int64_t windows = (p.num_tokens + a.window - 1) / a.window;
  const int64_t shares = (2 * p.num_heads + kWavesPerBlock - 1) / kWavesPerBlock;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(block_store_tags_kernel<CODEC, LDT, FORM>),
                     dim3(static_cast<uint32_t>(windows), static_cast<uint32_t>(shares), layers), dim3(kBlockThreads),
                     0, stream, a);
  return hipGetLastError();
}

template <int CODEC, int LDT>
hipError_t launch_typed(const BlockStoreParams& p, hipStream_t stream) {
  const int64_t elt = LDT == kLinF32 ? 4 : 2;
  uint64_t all = static_cast<uint64_t>(p.lin_token_stride * elt) | static_cast<uint64_t>(p.head_dim * elt) |
                 static_cast<uint64_t>(p.num_layers > 1 ? p.lin_layer_stride * elt : 0) |
                 static_cast<uint64_t>(p.block_size);
  for (int kv = 0; kv < 2; ++kv)
    all |= reinterpret_cast<uint64_t>(p.lin[kv]) | reinterpret_cast<uint64_t>(p.cache[kv]) |
           static_cast<uint64_t>(p.block_stride[kv]) | static_cast<uint64_t>(p.num_layers > 1 ? p.layer_stride[kv] : 0);
  if (all % 16 != 0 || p.head_dim % 8 != 0) return launch_form<CODEC, LDT, kElements>(p, stream);
  if (p.head_dim <= 128) {
    if (p.block_size == 16) return launch_form<CODEC, LDT, kHeldPieces>(p, stream);
    if (p.block_size == 32) return launch_form<CODEC, LDT, kHeldPieces2>(p, stream);
    if (p.block_size == 64) return launch_form<CODEC, LDT, kHeldPieces4>(p, stream);
  }
  return launch_form<CODEC, LDT, kPieces>(p, stream);
}

template <int CODEC>
hipError_t launch_codec(const BlockStoreParams& p, hipStream_t stream) {
  switch (p.lin_dtype) {
    case kLinF32: return launch_typed<CODEC, kLinF32>(p, stream);
    case kLinF16: return launch_typed<CODEC, kLinF16>(p, stream);
    case kLinBF16: return launch_typed<CODEC, kLinBF16>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_block_store(const BlockStoreParams& p, hipStream_t stream) {
  if (p.owner == nullptr && (p.num_tokens > kStoreScanTokens || p.block_size > kStoreScanColumns)) return hipErrorInvalidValue;
  return p.codec == kE4M3 ? launch_codec<kE4M3>(p, stream)
         : p.codec == kE5M2 ? launch_codec<kE5M2>(p, stream) : hipErrorInvalidValue;
}

hipError_t launch_block_tag_reset(const int64_t* slots, int64_t n, int64_t num_blocks, int64_t block_size,
                                  uint64_t* owner, hipStream_t stream) {
  const int64_t groups = (n * block_size + kBlockThreads - 1) / kBlockThreads;
  if (groups < 1 || groups >= int64_t{1} << 31) return hipErrorInvalidValue;
  hipLaunchKernelGGL(block_tag_reset_kernel, dim3(static_cast<uint32_t>(groups)), dim3(kBlockThreads), 0, stream, slots,
                     n, num_blocks, block_size, owner);
  return hipGetLastError();
}

}  // namespace kvhip
