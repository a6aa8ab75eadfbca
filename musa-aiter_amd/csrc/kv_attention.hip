// Attention over a paged FP8 cache with one scale per (block, head): kv_paged_attention_fp8.
//
//   s_j = softmax_scale * ks[blk(j), h] * sum_d q_d decode(K[blk(j), h, d, j % bs])
//   o_d = sum_j e^(s_j - lse) vs[blk(j), h] decode(V[blk(j), h, d, j % bs]),  lse = log sum_j e^(s_j)
//
// over the positions j that the row sees.  One pass over the cache with a running maximum and sum in base 2
// (p_j = 2^(s_j log2(e) - m)); parts of a sequence that run side by side leave (m, l, acc) in a workspace and
// a second launch joins them.
#include "kv_serving.h"

namespace kvhip {
namespace {

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

// Cached tokens of sequence b that its table has room for.
__device__ __forceinline__ int64_t seq_len(const AttnCall& c, int64_t b) { return int_at(c.lens, b, c.wide_lens); }

__device__ __forceinline__ int64_t table_block(const AttnCall& c, int64_t b, int64_t j) {
  return int_at(c.tables, b * c.table_stride + j, c.wide_tables);
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

// Partial results of split s: m and l at [s, row, head], then acc at [s, row, head, dim].
__device__ __forceinline__ float* part_ml(const AttnCall& c, int64_t s, int64_t rh) {
  return static_cast<float*>(c.workspace) + 2 * (s * c.rows * c.heads + rh);
}
__device__ __forceinline__ float* part_acc(const AttnCall& c, int64_t s, int64_t rh) {
  return static_cast<float*>(c.workspace) + 2 * c.splits * c.rows * c.heads + (s * c.rows * c.heads + rh) * c.head_dim;
}

// Tokens of a part start at multiples of this.
constexpr int64_t kPartTokens = 64;

struct Span {
  int64_t lo, hi;
};

// Part s of the positions [lo, hi).
__device__ __forceinline__ Span part_span(int64_t lo, int64_t hi, int64_t s, int64_t splits) {
  lo = lo / kPartTokens * kPartTokens;
  if (hi <= lo) return {lo, lo};
  const int64_t tiles = (hi - lo + kPartTokens - 1) / kPartTokens;
  const int64_t per = (tiles + splits - 1) / splits * kPartTokens;
  const int64_t from = lo + s * per;
  const int64_t to = from + per;
  return {from < hi ? from : hi, to < hi ? to : hi};
}

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

  // The sequence of this row.
  int64_t seq = -1, pos = -1, len = 0;
  if (c.starts == nullptr) {
    seq = t < c.batch ? t : -1;
    if (seq >= 0) {
      len = seq_len(c, seq);
      pos = len - 1;
    }
  } else {
    for (int64_t b0 = 0; b0 < c.batch && seq < 0; b0 += kWave) {
      const int64_t b = b0 + lane;
      SeqRows r{0, 0};
      if (b < c.batch) r = seq_rows(c, b);
      const uint64_t hit = ballot(r.count > 0 && t >= r.first && t < r.first + r.count);
      if (hit != 0) {
        const int src = __builtin_ctzll(hit);
        seq = b0 + src;
        len = seq_len(c, seq);
        pos = len - readlane64(r.count, src) + (t - readlane64(r.first, src));
      }
    }
  }
  if (seq < 0) {
    if (!c.fill_rows || split != 0) return;
    for (int64_t d = threadIdx.x; d < c.head_dim; d += kBlockThreads) store_o<DT>(c.out, rh * c.head_dim + d, 0.0f);
    if (c.lse != nullptr && threadIdx.x == 0) c.lse[rh] = -__builtin_inff();
    return;
  }
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
    if (c.splits > 1) part_acc(c, split, rh)[d] = o;
    else store_o<DT>(c.out, rh * c.head_dim + d, sum == 0.0f ? 0.0f : o / sum);
  }
  if (threadIdx.x == 0) {
    if (c.splits > 1) {
      part_ml(c, split, rh)[0] = top;
      part_ml(c, split, rh)[1] = sum;
    } else if (c.lse != nullptr) {
      c.lse[rh] = sum == 0.0f ? -__builtin_inff() : (top + log2f(sum)) * kLn2;
    }
  }
}

// ----- joining the parts: one wave per (row, head) -------------------------------------------------
template <int DT>
__global__ __launch_bounds__(kBlockThreads) void attention_join_kernel(const AttnCall c) {
  const int64_t rh = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave_in_block();
  if (rh >= c.rows * c.heads) return;
  const int64_t t = rh / c.heads;
  if (c.starts != nullptr) {  // rows of no sequence have no parts
    bool mine = false;
    for (int64_t b0 = 0; b0 < c.batch && !mine; b0 += kWave) {
      SeqRows r{0, 0};
      if (b0 + lane_id() < c.batch) r = seq_rows(c, b0 + lane_id());
      mine = ballot(t >= r.first && t < r.first + r.count) != 0;
    }
    if (!mine) return;
  } else if (t >= c.batch) {
    return;
  }
  float top = -__builtin_inff();
  for (int64_t s = 0; s < c.splits; ++s) top = fmaxf(top, part_ml(c, s, rh)[0]);
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  float sum = 0.0f;
  for (int64_t s = 0; s < c.splits; ++s) sum += part_ml(c, s, rh)[1] * __builtin_amdgcn_exp2f(part_ml(c, s, rh)[0] - ref);
  for (int64_t d = lane_id(); d < c.head_dim; d += kWave) {
    float o = 0.0f;
    for (int64_t s = 0; s < c.splits; ++s)
      o += part_acc(c, s, rh)[d] * __builtin_amdgcn_exp2f(part_ml(c, s, rh)[0] - ref);
    store_o<DT>(c.out, rh * c.head_dim + d, sum == 0.0f ? 0.0f : o / sum);
  }
  if (c.lse != nullptr && lane_id() == 0) c.lse[rh] = sum == 0.0f ? -__builtin_inff() : (top + log2f(sum)) * kLn2;
}

template <int DT>
hipError_t launch_join(const AttnCall& c, hipStream_t stream) {
  const int64_t groups = (c.rows * c.heads + kWavesPerBlock - 1) / kWavesPerBlock;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_join_kernel<DT>), dim3(static_cast<uint32_t>(groups)),
                     dim3(kBlockThreads), 0, stream, c);
  return hipGetLastError();
}

template <int DT, int CODEC>
hipError_t launch_any(const AttnCall& c, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(c.rows), static_cast<uint32_t>(c.heads), static_cast<uint32_t>(c.splits));
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_any_kernel<DT, CODEC>), grid, dim3(kBlockThreads), 0, stream, c);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_dtype(const AttnCall& c, hipStream_t stream) {
  const hipError_t err = c.codec == kE4M3 ? launch_any<DT, kE4M3>(c, stream) : launch_any<DT, kE5M2>(c, stream);
  if (err != hipSuccess || c.splits == 1) return err;
  return launch_join<DT>(c, stream);
}

}  // namespace

int64_t attention_splits(const AttnCall& c, int64_t longest) {
  const int64_t groups = c.rows * c.heads;
  int64_t splits = groups > 0 ? 1024 / groups : 1;
  const int64_t most = longest / 256;
  splits = splits < most ? splits : most;
  return splits < 1 ? 1 : splits > 64 ? 64 : splits;
}

int64_t attention_workspace(const AttnCall& c) {
  return c.splits <= 1 ? 0 : 4 * c.splits * c.rows * c.heads * (c.head_dim + 2);
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
