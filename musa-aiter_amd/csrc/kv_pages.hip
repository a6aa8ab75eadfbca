// Bookkeeping of a paged cache's pages: free, fork, extend (with copies of shared pages) and compact.
//
// A sequence owns the first ceil(len / block_size) entries of its table row; refs[p] counts the rows (and
// whatever else the caller counts) that own page p, and 0 means free.  Everything is decided on the device:
// the host reads nothing, so the calls can be captured.  Which page goes where depends on the tables alone
// (free pages are taken lowest id first, rows in order), never on the order in which waves run: the only
// atomics are integer additions to reference counts.
//
// What bounds them: the decisions are a prefix sum over the rows and one over the pages, made by one workgroup
// (a second launch moves the pages over the whole chip); with no page to move a call is launch latency.
#include "kv_serving.h"

namespace kvhip {
namespace {

using i32x4 = int32_t __attribute__((ext_vector_type(4)));

constexpr int kScanThreads = 1024;
constexpr int kScanWaves = kScanThreads / kWave;
constexpr int kPerThread = 8;                               // pages a thread looks at per step of a scan
constexpr int64_t kScanStep = kScanThreads * kPerThread;

// Header of the workspace, then the arrays (all int64).
struct PagesHeader {
  int64_t moves;   // pairs in src / dst
  int64_t fits;    // extend: whether anything was done
  int64_t live;    // compact: pages in use
  int64_t unused;
};
constexpr int64_t kHeaderWords = sizeof(PagesHeader) / 8;

struct PagesArgs {
  musa_aiter_hip_pages_call c;
  PagesHeader* head;
  int64_t* src;      // moved pages
  int64_t* dst;
  int64_t* a;        // fork: new rows; extend: first need of each row; compact: new id of pages >= live
  int64_t* b;        // fork: new lengths
  int64_t* list;     // extend: free pages taken
};

__device__ __forceinline__ int64_t row_value(const musa_aiter_hip_pages_call& c, int64_t b) {
  return c.wide_rows ? static_cast<const int64_t*>(c.rows)[b] : static_cast<const int32_t*>(c.rows)[b];
}

// (In this form no length, however wrong, runs past int64.)
__device__ __forceinline__ int64_t pages_of(int64_t len, int64_t bs) { return len <= 0 ? 0 : (len - 1) / bs + 1; }

// Entries of a row that its length covers (a length past the row's end owns the whole row).
__device__ __forceinline__ int64_t owned_of(const musa_aiter_hip_pages_call& c, int64_t len) {
  const int64_t n = pages_of(len, c.block_size);
  return n < c.max_blocks ? n : c.max_blocks;
}

template <typename IT>
__device__ __forceinline__ void add_ref(IT* refs, int64_t page, int by) {
  if constexpr (sizeof(IT) == 8)
    atomicAdd(reinterpret_cast<unsigned long long*>(refs + page), static_cast<unsigned long long>(static_cast<int64_t>(by)));
  else
    atomicAdd(reinterpret_cast<int*>(refs + page), by);
}

// Exclusive prefix sum over the workgroup's threads; *total is the sum.  `part` holds kScanWaves values.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* part, int64_t* total) {
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t y = __shfl_up(static_cast<long long>(x), o);
    if (lane_id() >= o) x += y;
  }
  __syncthreads();  // the last call's readers of part are done
  if (lane_id() == kWave - 1) part[threadIdx.x >> 6] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int w = 0; w < kScanWaves; ++w) {
    const int64_t y = part[w];
    if (w < static_cast<int>(threadIdx.x >> 6)) before += y;
    all += y;
  }
  *total = all;
  return before + x - v;
}

// ----- free: one workgroup per row --------------------------------------------------------------
template <typename IT>
__global__ __launch_bounds__(kBlockThreads) void pages_free_kernel(const musa_aiter_hip_pages_call c) {
  const int64_t b = blockIdx.x;
  IT* lens = static_cast<IT*>(c.lens);
  IT* refs = static_cast<IT*>(c.refs);
  IT* row = static_cast<IT*>(c.tables) + b * c.table_stride;
  const int64_t len = lens[b], asked = row_value(c, b);
  const int64_t keep = asked < 0 || asked > len ? len : asked;
  const int64_t last = owned_of(c, len);
  for (int64_t j = pages_of(keep, c.block_size) + threadIdx.x; j < last; j += kBlockThreads) {
    const int64_t page = row[j];
    if (page >= 0 && page < c.num_blocks) add_ref(refs, page, -1);
    row[j] = -1;
  }
  __syncthreads();  // every wave has read the length
  if (threadIdx.x == 0 && keep != len) lens[b] = static_cast<IT>(keep);
}

// ----- fork: the new rows aside with the counts' changes, then into place -------------------------
template <typename IT, bool PLACE>
__global__ __launch_bounds__(kBlockThreads) void pages_fork_kernel(const PagesArgs a) {
  const musa_aiter_hip_pages_call& c = a.c;
  const int64_t b = blockIdx.x;
  const int64_t parent = row_value(c, b);
  if (parent == b) return;  // the row stays as it is
  IT* lens = static_cast<IT*>(c.lens);
  IT* refs = static_cast<IT*>(c.refs);
  IT* tables = static_cast<IT*>(c.tables);
  IT* aside = reinterpret_cast<IT*>(a.a) + b * c.max_blocks;
  if constexpr (PLACE) {
    for (int64_t j = threadIdx.x; j < c.max_blocks; j += kBlockThreads) tables[b * c.table_stride + j] = aside[j];
    if (threadIdx.x == 0) lens[b] = static_cast<IT>(a.b[b]);
  } else {
    const bool has = parent >= 0 && parent < c.batch;
    const int64_t len = has ? static_cast<int64_t>(lens[parent]) : 0;
    const int64_t gain = owned_of(c, len), loss = owned_of(c, lens[b]);
    for (int64_t j = threadIdx.x; j < c.max_blocks; j += kBlockThreads) {
      const int64_t now = has ? static_cast<int64_t>(tables[parent * c.table_stride + j]) : -1;
      const int64_t old = tables[b * c.table_stride + j];
      const bool takes = j < gain && now >= 0 && now < c.num_blocks;
      const bool drops = j < loss && old >= 0 && old < c.num_blocks;
      if (!(takes && drops && now == old)) {
        if (takes) add_ref(refs, now, 1);
        if (drops) add_ref(refs, old, -1);
      }
      aside[j] = static_cast<IT>(now);
    }
    if (threadIdx.x == 0) a.b[b] = len;
  }
}

// ----- extend -----------------------------------------------------------------------------------
// Rows take pages in order: first the copy of a shared partial last page, then the pages of the new tokens.
// A page that r owners share is copied by all the rows that grow into it but the last, and by all of them if
// somebody else owns it too: row b copies iff fewer than r - 1 rows before it grow into the same page.
template <typename IT>
constexpr int64_t kMostTokens = sizeof(IT) == 8 ? INT64_MAX : INT32_MAX;  // that a row's length can say

template <typename IT>
struct ExtendRow {
  int64_t len, grow, had, has, last;
  bool open;  // grows into a partial last page

  __device__ ExtendRow(const musa_aiter_hip_pages_call& c, int64_t b) {
    len = static_cast<const IT*>(c.lens)[b];
    len = len < 0 ? 0 : len > INT64_MAX / 2 ? INT64_MAX / 2 : len;  // such a row outgrows every table
    grow = row_value(c, b);
    grow = grow < 0 ? 0 : grow > c.max_new ? c.max_new : grow;
    had = pages_of(len, c.block_size);
    has = pages_of(len + grow, c.block_size);
    open = false;
    last = -1;
    if (grow > 0 && len % c.block_size != 0 && had <= c.max_blocks) {
      last = static_cast<const IT*>(c.tables)[b * c.table_stride + had - 1];
      open = last >= 0 && last < c.num_blocks;
    }
  }
};

template <typename IT>
__global__ __launch_bounds__(kScanThreads) void pages_extend_kernel(const PagesArgs a) {
  const musa_aiter_hip_pages_call& c = a.c;
  IT* refs = static_cast<IT*>(c.refs);
  __shared__ int64_t part[kScanWaves];
  __shared__ alignas(16) int32_t grown[kScanThreads];  // partial last page that a row grows into, or -1
  __shared__ int too_long, shared_pages;
  if (threadIdx.x == 0) too_long = 0;
  // What every row needs, and the sum in front of it.
  int64_t need_all = 0;
  for (int64_t base = 0; base < c.batch; base += kScanThreads) {
    const int64_t b = base + threadIdx.x;
    int64_t need = 0, owners = 0;
    int32_t last = -1;
    __syncthreads();  // the last round's flag has been read
    if (threadIdx.x == 0) shared_pages = 0;
    __syncthreads();
    if (b < c.batch) {
      const ExtendRow<IT> r(c, b);
      if (r.has > c.max_blocks || r.len + r.grow > kMostTokens<IT>) too_long = 1;
      need = r.has - r.had;
      if (r.open) {
        last = static_cast<int32_t>(r.last);
        owners = refs[r.last];
        if (owners > 1) shared_pages = 1;
      }
    }
    __syncthreads();
    bool copy = false;
    if (shared_pages) {
      int64_t earlier = 0;
      for (int64_t from = 0; from <= base; from += kScanThreads) {
        int32_t theirs = last;
        if (from < base) {
          const ExtendRow<IT> x(c, from + threadIdx.x);
          theirs = x.open ? static_cast<int32_t>(x.last) : -1;
        }
        __syncthreads();
        grown[threadIdx.x] = theirs;
        __syncthreads();
        const int until = from < base ? kScanThreads : static_cast<int>(threadIdx.x);
        if (owners > 1) {
          int o = 0;
#pragma unroll 4
          for (; o + 4 <= until; o += 4) {
            const i32x4 g = *reinterpret_cast<const i32x4*>(grown + o);
            earlier += (g[0] == last) + (g[1] == last) + (g[2] == last) + (g[3] == last);
          }
          for (; o < until; ++o) earlier += grown[o] == last;
        }
      }
      copy = owners > 1 && earlier < owners - 1;
    }
    need += copy;
    int64_t sum;
    const int64_t before = need_all + block_scan(need, part, &sum);
    if (b < c.batch) a.a[b] = 2 * before + copy;
    need_all += sum;
  }
  // The free pages, lowest first.
  int64_t free_all = 0;
  for (int64_t base = 0; base < c.num_blocks; base += kScanStep) {
    const int64_t p0 = base + static_cast<int64_t>(threadIdx.x) * kPerThread;
    uint32_t mask = 0;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (p0 + k < c.num_blocks && refs[p0 + k] == 0) mask |= 1u << k;
    int64_t sum;
    int64_t at = free_all + block_scan(__popc(mask), part, &sum);
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (mask >> k & 1) {
        if (at < need_all) a.list[at] = p0 + k;
        ++at;
      }
    free_all += sum;
  }
  __syncthreads();  // the list and every row's need are written, and too_long is
  const bool fits = need_all <= free_all && !too_long;
  if (threadIdx.x == 0) {
    a.head->fits = fits;
    *c.result = too_long ? -(int64_t{1} << 62) : free_all - need_all;
  }
  // The copies' pairs, in the rows' order.
  int64_t moves = 0;
  for (int64_t base = 0; base < c.batch; base += kScanThreads) {
    const int64_t b = base + threadIdx.x;
    const bool copy = fits && b < c.batch && (a.a[b] & 1);
    int64_t sum;
    const int64_t at = moves + block_scan(copy, part, &sum);
    if (copy) {
      const ExtendRow<IT> r(c, b);
      a.src[at] = r.last;
      a.dst[at] = a.list[a.a[b] >> 1];
    }
    moves += sum;
  }
  if (threadIdx.x == 0) a.head->moves = moves;
}

// ----- compact ----------------------------------------------------------------------------------
template <typename IT>
__global__ __launch_bounds__(kScanThreads) void pages_compact_kernel(const PagesArgs a) {
  const musa_aiter_hip_pages_call& c = a.c;
  IT* refs = static_cast<IT*>(c.refs);
  __shared__ int64_t part[kScanWaves];
  int64_t live = 0;
  {
    int64_t mine = 0;
    for (int64_t p = threadIdx.x; p < c.num_blocks; p += kScanThreads) mine += refs[p] > 0;
    block_scan(mine, part, &live);
  }
  // Holes below `live` and pages in use from there on: as many of the one as of the other.
  int64_t holes = 0, movers = 0;
  for (int64_t base = 0; base < c.num_blocks; base += kScanStep) {
    const int64_t p0 = base + static_cast<int64_t>(threadIdx.x) * kPerThread;
    uint32_t hole = 0, mover = 0;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (p0 + k < c.num_blocks) {
        const bool used = refs[p0 + k] > 0;
        if (p0 + k < live) hole |= static_cast<uint32_t>(!used) << k;
        else {
          mover |= static_cast<uint32_t>(used) << k;
          a.a[p0 + k] = p0 + k;
        }
      }
    int64_t sum;
    int64_t at = holes + block_scan(__popc(hole), part, &sum);
    holes += sum;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (hole >> k & 1) a.dst[at++] = p0 + k;
    at = movers + block_scan(__popc(mover), part, &sum);
    movers += sum;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (mover >> k & 1) a.src[at++] = p0 + k;
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < movers; i += kScanThreads) {
    const int64_t from = a.src[i], to = a.dst[i];
    a.a[from] = to;
    refs[to] = refs[from];
    refs[from] = 0;
  }
  if (threadIdx.x == 0) {
    a.head->moves = movers;
    a.head->live = live;
    *c.result = live;
  }
}

// ----- the second launch: pages move, and what follows from the tables -----------------------------
// A workgroup takes (pair, layer, plane) items in turn; VEC is the width every address allows.
template <int VEC>
__device__ __forceinline__ void move_pages(const PagesArgs& a) {
  const musa_aiter_hip_pages_call& c = a.c;
  const int64_t items = a.head->moves * c.layers * 2;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t pair = it / (2 * c.layers);
    const int64_t rem = it - pair * 2 * c.layers;
    const int64_t layer = rem >> 1;
    const int kv = static_cast<int>(rem & 1);
    const int64_t src = a.src[pair], dst = a.dst[pair];
    uint8_t* plane = static_cast<uint8_t*>(c.cache[kv]) + layer * c.layer_stride[kv];
    const uint8_t* from = plane + src * c.block_stride[kv];
    uint8_t* to = plane + dst * c.block_stride[kv];
    const int64_t step = static_cast<int64_t>(kBlockThreads) * VEC;
    int64_t at = static_cast<int64_t>(threadIdx.x) * VEC;
    for (; at + 3 * step + VEC <= c.block_bytes; at += 4 * step) {
      typename VecType<VEC>::T v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = ldv<VEC>(from + at + k * step);
#pragma unroll
      for (int k = 0; k < 4; ++k) stv<VEC>(to + at + k * step, v[k]);
    }
    for (; at + VEC <= c.block_bytes; at += step) stv<VEC>(to + at, ldv<VEC>(from + at));
    if (c.scale[kv] != nullptr) {
      float* s = c.scale[kv] + layer * c.num_blocks * c.scale_values;
      for (int64_t h = threadIdx.x; h < c.scale_values; h += kBlockThreads)
        s[dst * c.scale_values + h] = s[src * c.scale_values + h];
    }
  }
}

// The rows, a workgroup each (one after the other by the scan's single workgroup they took 15 us for 128 rows), and
// the copies.
template <typename IT, int VEC>
__global__ __launch_bounds__(kBlockThreads) void pages_extend_finish_kernel(const PagesArgs a) {
  const musa_aiter_hip_pages_call& c = a.c;
  IT* lens = static_cast<IT*>(c.lens);
  IT* refs = static_cast<IT*>(c.refs);
  const bool fits = a.head->fits != 0;
  for (int64_t b = blockIdx.x; b < c.batch; b += gridDim.x) {
    const ExtendRow<IT> r(c, b);
    const int64_t grow = fits ? r.grow : 0;
    const int64_t first = a.a[b] >> 1;
    const int copy = static_cast<int>(a.a[b] & 1);
    __syncthreads();  // every wave has read the row
    IT* row = static_cast<IT*>(c.tables) + b * c.table_stride;
    if (grow > 0) {
      if (threadIdx.x == 0) {
        if (copy) {
          const int64_t page = a.list[first];
          add_ref(refs, r.last, -1);
          refs[page] = 1;
          row[r.had - 1] = static_cast<IT>(page);
        }
        lens[b] = static_cast<IT>(r.len + grow);
      }
      for (int64_t j = r.had + threadIdx.x; j < r.has; j += kBlockThreads) {
        const int64_t page = a.list[first + copy + j - r.had];
        refs[page] = 1;
        row[j] = static_cast<IT>(page);
      }
    }
    for (int64_t k = threadIdx.x; k < c.max_new; k += kBlockThreads) {
      int64_t slot = -1;
      if (k < grow) {
        const int64_t pos = r.len + k, j = pos / c.block_size;
        const int64_t page = j >= r.had ? a.list[first + copy + j - r.had] : copy ? a.list[first] : r.open ? r.last : -1;
        if (page >= 0) slot = page * c.block_size + (pos - j * c.block_size);
      }
      c.slots[b * c.max_new + k] = slot;
    }
  }
  move_pages<VEC>(a);
}

template <typename IT, int VEC>
__global__ __launch_bounds__(kBlockThreads) void pages_compact_finish_kernel(const PagesArgs a) {
  const musa_aiter_hip_pages_call& c = a.c;
  if (a.head->moves > 0) {
    const int64_t live = a.head->live;
    const int64_t threads = static_cast<int64_t>(gridDim.x) * kBlockThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlockThreads + threadIdx.x; i < c.batch * c.max_blocks;
         i += threads) {
      const int64_t b = i / c.max_blocks;
      IT* entry = static_cast<IT*>(c.tables) + b * c.table_stride + (i - b * c.max_blocks);
      const int64_t page = *entry;
      if (page >= live && page < c.num_blocks) *entry = static_cast<IT>(a.a[page]);
    }
  }
  move_pages<VEC>(a);
}

int copy_width(const musa_aiter_hip_pages_call& c) {
  uint64_t all = static_cast<uint64_t>(c.block_bytes);
  for (int kv = 0; kv < 2; ++kv)
    all |= reinterpret_cast<uint64_t>(c.cache[kv]) | static_cast<uint64_t>(c.block_stride[kv]) |
           static_cast<uint64_t>(c.layer_stride[kv]);
  return all % 16 == 0 ? 16 : 1;
}

// Workgroups of a second launch: enough for every item of `most` moved pages, at most eight per CU.
uint32_t finish_groups(const musa_aiter_hip_pages_call& c, int64_t most, int64_t entries) {
  int64_t n = most * c.layers * 2;
  const int64_t e = (entries + kBlockThreads - 1) / kBlockThreads;
  n = n > e ? n : e;
  return static_cast<uint32_t>(n < 1 ? 1 : n > 2048 ? 2048 : n);
}

PagesArgs lay_out(const musa_aiter_hip_pages_call& c, PagesKind kind) {
  PagesArgs a{};
  a.c = c;
  a.head = static_cast<PagesHeader*>(c.workspace);
  int64_t* p = static_cast<int64_t*>(c.workspace) + kHeaderWords;
  if (kind == kPagesFork) {
    a.b = p;
    a.a = p + c.batch;
  } else if (kind == kPagesExtend) {
    a.src = p;
    a.dst = a.src + c.batch;
    a.a = a.dst + c.batch;
    a.list = a.a + c.batch;
  } else {
    a.src = p;
    a.dst = a.src + c.num_blocks;
    a.a = a.dst + c.num_blocks;
  }
  return a;
}

template <typename IT>
hipError_t launch_typed(const musa_aiter_hip_pages_call& c, PagesKind kind, hipStream_t stream) {
  const uint32_t rows = static_cast<uint32_t>(c.batch);
  const dim3 threads(kBlockThreads);
  if (kind == kPagesFree) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(pages_free_kernel<IT>), dim3(rows), threads, 0, stream, c);
    return hipGetLastError();
  }
  const PagesArgs a = lay_out(c, kind);
  if (kind == kPagesFork) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(pages_fork_kernel<IT, false>), dim3(rows), threads, 0, stream, a);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(pages_fork_kernel<IT, true>), dim3(rows), threads, 0, stream, a);
    return hipGetLastError();
  }
  const bool wide_copy = copy_width(c) == 16;
  if (kind == kPagesExtend) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(pages_extend_kernel<IT>), dim3(1), dim3(kScanThreads), 0, stream, a);
    const dim3 grid(finish_groups(c, c.batch, c.batch));
    if (wide_copy)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(pages_extend_finish_kernel<IT, 16>), grid, threads, 0, stream, a);
    else
      hipLaunchKernelGGL(HIP_KERNEL_NAME(pages_extend_finish_kernel<IT, 1>), grid, threads, 0, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(HIP_KERNEL_NAME(pages_compact_kernel<IT>), dim3(1), dim3(kScanThreads), 0, stream, a);
  const dim3 grid(finish_groups(c, c.num_blocks, c.batch * c.max_blocks));
  if (wide_copy)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(pages_compact_finish_kernel<IT, 16>), grid, threads, 0, stream, a);
  else
    hipLaunchKernelGGL(HIP_KERNEL_NAME(pages_compact_finish_kernel<IT, 1>), grid, threads, 0, stream, a);
  return hipGetLastError();
}

}  // namespace

int64_t pages_workspace(const musa_aiter_hip_pages_call& c, PagesKind kind) {
  int64_t words = kHeaderWords;
  if (kind == kPagesFork) words += c.batch + (c.batch * c.max_blocks * (c.wide ? 8 : 4) + 7) / 8;
  else if (kind == kPagesExtend) words += 3 * c.batch + c.num_blocks;
  else if (kind == kPagesCompact) words += 3 * c.num_blocks;
  else return 0;
  return 8 * words;
}

hipError_t launch_pages(const musa_aiter_hip_pages_call& c, PagesKind kind, hipStream_t stream) {
  const int64_t most = int64_t{1} << 31;
  if (c.batch < 0 || c.batch >= most || c.max_blocks < 0 || c.max_blocks >= most || c.num_blocks < 0 ||
      c.num_blocks >= most || c.block_size < 1 || c.max_new < 0 || c.max_new >= most)
    return hipErrorInvalidValue;
  const bool needs_rows = c.batch > 0;
  if (needs_rows && c.max_blocks > 0 && c.tables == nullptr) return hipErrorInvalidValue;
  if (c.num_blocks > 0 && c.refs == nullptr) return hipErrorInvalidValue;
  if (kind != kPagesCompact && needs_rows && (c.lens == nullptr || c.rows == nullptr)) return hipErrorInvalidValue;
  if (kind != kPagesFree && (c.workspace == nullptr || c.workspace_bytes < pages_workspace(c, kind)))
    return hipErrorInvalidValue;
  if (kind == kPagesExtend || kind == kPagesCompact) {
    if (c.result == nullptr || c.layers < 0 || c.block_bytes < 0 || c.scale_values < 0) return hipErrorInvalidValue;
    if (c.layers > 0 && c.block_bytes > 0 && (c.cache[0] == nullptr || c.cache[1] == nullptr)) return hipErrorInvalidValue;
    if (kind == kPagesExtend && c.batch * c.max_new > 0 && c.slots == nullptr) return hipErrorInvalidValue;
  } else if (!needs_rows) {
    return hipSuccess;
  }
  return c.wide ? launch_typed<int64_t>(c, kind, stream) : launch_typed<int32_t>(c, kind, stream);
}

}  // namespace kvhip
