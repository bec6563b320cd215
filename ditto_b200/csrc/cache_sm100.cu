// Kernels of the paged key/value cache: appending, and the page operations.
#include "cache_sm100.cuh"

#include "host_util.cuh"
#include "masked_sm100.cuh"
#include "sm100_ptx.cuh"

namespace ditto_b200 {
namespace cache {
namespace {

constexpr int kAppendThreads = 256;

// A thread a 16-byte piece of a key row and of the value row beside it.  Bound by the bytes, each read once and written once, and below some MB
// by latency: 4 us for 64 tokens of 8 heads, 6 us for 8192 of two.
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int per_token = p.kv_heads * p.pieces;
  const long long total = static_cast<long long>(p.tokens) * per_token;
  for (long long i = static_cast<long long>(blockIdx.x) * kAppendThreads + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * kAppendThreads) {
    const int token = static_cast<int>(i / per_token), rest = static_cast<int>(i - static_cast<long long>(token) * per_token);
    const int head = rest / p.pieces, piece = rest - head * p.pieces;
    int seq = token, first = token, end = token + 1;
    if (p.starts != nullptr) {
      int lo = 0, hi = p.batch;                    // the last sequence that starts at or before the token
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.starts[mid] <= token) lo = mid;
        else hi = mid;
      }
      seq = lo;
      first = p.starts[seq];
      end = p.starts[seq + 1];
      if (token < first || token >= end) continue;          // in front of the first sequence, or behind the last
    }
    const int at = p.lengths[seq] - (end - first) + (token - first);
    int id = -1;
    if (at >= 0 && at / p.page < p.table_cols) id = p.table[seq * p.table_stride + at / p.page];
    if (id < 0 || id >= p.pages) {
      if (p.status != nullptr) atomicCAS(p.status, 0, masked::kBadPage);
      continue;
    }
    const int slot = at % p.page;
    const uint4 k = *reinterpret_cast<const uint4*>(p.keys + token * p.k_token + head * p.k_head + piece * 16);
    const uint4 v = *reinterpret_cast<const uint4*>(p.values + token * p.v_token + head * p.v_head + piece * 16);
    *reinterpret_cast<uint4*>(p.key_pages + id * p.kp_page + slot * p.kp_slot + head * p.kp_head + piece * 16) = k;
    *reinterpret_cast<uint4*>(p.value_pages + id * p.vp_page + slot * p.vp_slot + head * p.vp_head + piece * 16) = v;
  }
}

// ------------------------------------------------------------------ page copies
constexpr int kCopyThreads = 512, kCopyUnroll = 4;

// What a fork and a compaction do to the tables beside their copies, dealt out over the CTAs of the copy (a launch less each).
// The child's row of pair i, and one reference more for every page in it: a CTA a pair.
__device__ __forceinline__ void share_pages(const TableJob& job, const Tables& t, int n) {
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int parent = job.parents[i], child = job.children[i];
    if (parent < 0 || parent >= t.sequences || child < 0 || child >= t.sequences || parent == child) continue;
    const long long length = min(static_cast<long long>(max(0, t.lengths[parent])), static_cast<long long>(t.cols) * t.page);
    const int full = static_cast<int>(length / t.page), last = job.target[i];
    for (int k = threadIdx.x; k < t.cols; k += blockDim.x) {
      const int page = k < full ? t.table[parent * t.stride + k] : k == full ? last : -1;
      t.table[child * t.stride + k] = page;
      if (page >= 0 && page < t.pages) atomicAdd(t.references + page, 1);
    }
    if (threadIdx.x == 0) t.lengths[child] = static_cast<int>(length);
  }
}
__device__ __forceinline__ void rename_pages(const TableJob& job, const Tables& t) {
  const long long total = static_cast<long long>(t.sequences) * t.cols, step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const long long s = i / t.cols, k = i - s * t.cols;
    const int page = t.table[s * t.stride + k];
    job.new_table[s * job.new_stride + k] = page >= 0 && page < t.pages ? job.renamed[page] : page;
  }
}

// The pieces of all pages to be copied, in all pools, dealt out evenly: one CTA takes runs of kCopyThreads * kCopyUnroll pieces, each thread
// with kCopyUnroll loads of 16 bytes in flight.  Bound by the bytes: read once, written once; 2000 pages compacted, 2.1 GB read and written, 348 us
// (6.2 TB/s).
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int n = p.n_device != nullptr ? min(*p.n_device, p.n) : p.n;
  if (p.job.parents != nullptr) share_pages(p.job, p.job.tables, n);
  if (p.job.renamed != nullptr) rename_pages(p.job, p.job.tables);
  constexpr int kRun = kCopyThreads * kCopyUnroll;
  const int runs = (p.pools.pieces + kRun - 1) / kRun;           // of a page in a pool
  const long long total = static_cast<long long>(n) * p.pools.count * runs;
  for (long long i = blockIdx.x; i < total; i += gridDim.x) {
    const int run = static_cast<int>(i % runs), pool = static_cast<int>(i / runs % p.pools.count), pair = static_cast<int>(i / runs / p.pools.count);
    const int from = p.source[pair], to = p.target[pair];
    if (from < 0 || to < 0 || from >= p.pages || to >= p.pages) {
      if ((from >= p.pages || to >= p.pages) && threadIdx.x == 0 && p.status != nullptr) atomicCAS(p.status, 0, masked::kBadPage);
      continue;
    }
    const uint4* src = reinterpret_cast<const uint4*>(p.pools.base[pool] + from * p.pools.stride);
    uint4* dst = reinterpret_cast<uint4*>(p.pools.base[pool] + to * p.pools.stride);
    uint4 v[kCopyUnroll];
    const int first = run * kRun + threadIdx.x;
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (first + u * kCopyThreads < p.pools.pieces) v[u] = src[first + u * kCopyThreads];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (first + u * kCopyThreads < p.pools.pieces) dst[first + u * kCopyThreads] = v[u];
  }
}

// ------------------------------------------------------------------ tables
constexpr int kTableThreads = 1024;

// Sum over the threads in front of this one, and of all; `scratch` holds a word a warp and one more.
__device__ __forceinline__ int block_scan(int v, int* scratch, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int x = scratch[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    scratch[lane] = x;
  }
  __syncthreads();
  *total = scratch[kTableThreads / 32 - 1];
  return (warp > 0 ? scratch[warp - 1] : 0) + incl - v;
}

// Calls found(k, page) for the k-th free page, lowest first, k < wanted; all threads of the CTA together.  Returns how many there are (at
// least, where it stopped early).
template <class Found>
__device__ __forceinline__ int free_pages(const int* references, int pages, int wanted, int* scratch, Found found) {
  int before = 0;
  for (int base = 0; base < pages && before < wanted; base += kTableThreads * 4) {
    int refs[4];
    const int first = base + static_cast<int>(threadIdx.x) * 4;
    int mine = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      refs[u] = first + u < pages ? references[first + u] : 1;
      mine += refs[u] <= 0;
    }
    int total;
    int k = before + block_scan(mine, scratch, &total);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (refs[u] <= 0) {
        if (k < wanted) found(k, first + u);
        ++k;
      }
    before += total;
  }
  return before;
}

// A CTA a sequence to be freed.  A sequence that is named twice is freed once.  Latency: 4 us.
__global__ void __launch_bounds__(256) free_kernel(const __grid_constant__ Tables t, const int* sequences, int n) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int s = sequences[blockIdx.x];
  if (s < 0 || s >= t.sequences) return;
  int again = 0;
  for (int i = threadIdx.x; i < static_cast<int>(blockIdx.x); i += blockDim.x) again |= sequences[i] == s;
  if (__syncthreads_or(again)) return;
  int* row = t.table + s * t.stride;
  for (int k = threadIdx.x; k < t.cols; k += blockDim.x) {
    const int page = row[k];
    if (page < 0) continue;
    row[k] = -1;
    if (page < t.pages) atomicSub(t.references + page, 1);       // (whole numbers: the order does not show)
    else if (t.status != nullptr) atomicCAS(t.status, 0, masked::kBadPage);
  }
  if (threadIdx.x == 0) t.lengths[s] = 0;
}

__global__ void __launch_bounds__(kTableThreads, 1) reserve_kernel(const __grid_constant__ Tables t, const int* counts, int* first) {
  __shared__ int scratch[kTableThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  // pages that each sequence needs more, and the number in front of it
  int needed = 0;
  bool fits = true;
  for (int base = 0; base < t.sequences; base += kTableThreads) {
    const int s = base + static_cast<int>(threadIdx.x);
    int need = 0;
    if (s < t.sequences) {
      const int count = max(0, counts[s]), have = (max(0, t.lengths[s]) + t.page - 1) / t.page;
      const long long want = (static_cast<long long>(max(0, t.lengths[s])) + count + t.page - 1) / t.page;
      if (want > t.cols) fits = false;
      else need = static_cast<int>(want) - have;
    }
    int total;
    const int at = needed + block_scan(need, scratch, &total);
    if (s < t.sequences) first[s] = at;
    needed += total;
  }
  if (threadIdx.x == 0) first[t.sequences] = needed;
  const int short_of_columns = __syncthreads_or(!fits);
  const int found = short_of_columns ? 0 : free_pages(t.references, t.pages, needed, scratch, [](int, int) {});
  if (short_of_columns || found < needed) {                     // all or nothing
    if (threadIdx.x == 0 && t.status != nullptr) atomicCAS(t.status, 0, masked::kNoPages);
    return;
  }
  __syncthreads();
  free_pages(t.references, t.pages, needed, scratch, [&](int k, int page) {
    int lo = 0, hi = t.sequences;                               // the sequence whose pages begin at or before k
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (first[mid] <= k) lo = mid;
      else hi = mid;
    }
    t.table[lo * t.stride + (max(0, t.lengths[lo]) + t.page - 1) / t.page + k - first[lo]] = page;
    t.references[page] = 1;
  });
  __syncthreads();
  for (int s = threadIdx.x; s < t.sequences; s += kTableThreads) t.lengths[s] = max(0, t.lengths[s]) + max(0, counts[s]);
}

// One CTA: which child gets which free page.  source / target of pair i: the last page of its parent and the child's, -1 where there is
// nothing to copy (a last page that is full, a pair out of range); *count: n, or 0 where there are too few free pages.  Latency of the scans: 6 us.
__global__ void __launch_bounds__(kTableThreads, 1) fork_pages_kernel(const __grid_constant__ Tables t, const int* parents, const int* children, int n,
                                                                      int* source, int* target, int* list, int* count) {
  __shared__ int scratch[kTableThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  int needed = 0;
  for (int base = 0; base < n; base += kTableThreads) {
    const int i = base + static_cast<int>(threadIdx.x);
    int from = -1;
    if (i < n) {
      const int parent = parents[i], child = children[i];
      if (parent >= 0 && parent < t.sequences && child >= 0 && child < t.sequences && parent != child) {
        const long long length = min(static_cast<long long>(max(0, t.lengths[parent])), static_cast<long long>(t.cols) * t.page);
        if (length % t.page != 0) from = t.table[parent * t.stride + length / t.page];
        if (from >= t.pages) {
          from = -1;
          if (t.status != nullptr) atomicCAS(t.status, 0, masked::kBadPage);
        }
      }
      source[i] = from;
    }
    int total;
    const int at = needed + block_scan(from >= 0, scratch, &total);
    if (i < n) target[i] = from >= 0 ? at : -1;                 // (its number among the pages to be taken)
    needed += total;
  }
  const int found = free_pages(t.references, t.pages, needed, scratch, [&](int k, int page) { list[k] = page; });
  __syncthreads();
  const bool enough = found >= needed;
  if (threadIdx.x == 0) {
    *count = enough ? n : 0;
    if (!enough && t.status != nullptr) atomicCAS(t.status, 0, masked::kNoPages);
  }
  if (!enough) return;
  for (int i = threadIdx.x; i < n; i += kTableThreads)
    if (target[i] >= 0) target[i] = list[target[i]];
}

// One CTA: the k-th live page behind the first n (n live pages) moves to the k-th free place among them.  Latency of the scans: 4 us for 200
// pages, 6 us for 2000.
__global__ void __launch_bounds__(kTableThreads, 1) compact_pages_kernel(const int* references, int pages, int* new_references, int* renamed, int* source,
                                                                         int* target, int* count) {
  __shared__ int scratch[kTableThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  int mine = 0, n, moves = 0, holes = 0;
  for (int i = threadIdx.x; i < pages; i += kTableThreads) mine += references[i] > 0;
  block_scan(mine, scratch, &n);
  for (int base = 0; base < pages; base += kTableThreads) {
    const int i = base + static_cast<int>(threadIdx.x);
    const bool live = i < pages && references[i] > 0, move = live && i >= n, hole = i < n && !live;
    int total;
    // both counts in one scan: a round has at most kTableThreads of either
    const int at = block_scan((move ? 1 : 0) + (hole ? 1 << 16 : 0), scratch, &total);
    if (move) source[moves + (at & 0xffff)] = i;
    if (hole) target[holes + (at >> 16)] = i;
    if (i < pages) renamed[i] = i;
    moves += total & 0xffff;
    holes += total >> 16;
  }
  if (threadIdx.x == 0) *count = moves;
  __syncthreads();
  // (references and new_references may be the same: what is read here is either a page's old count or its new one, as it should be)
  for (int i = threadIdx.x; i < pages; i += kTableThreads) {
    const int r = references[i];
    if (new_references != references && (i < n ? r > 0 : r <= 0)) new_references[i] = r;
  }
  for (int k = threadIdx.x; k < moves; k += kTableThreads) {
    const int from = source[k], to = target[k], r = references[from];
    renamed[from] = to;
    new_references[to] = r;
    new_references[from] = 0;
  }
}

cudaLaunchConfig_t config(unsigned grid, int threads, cudaStream_t stream, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

}  // namespace

cudaError_t launch_append(const AppendParams& p, cudaStream_t stream) {
  const long long total = static_cast<long long>(p.tokens) * p.kv_heads * p.pieces, ctas = (total + kAppendThreads - 1) / kAppendThreads;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = config(static_cast<unsigned>(ctas < 148 * 16 ? ctas : 148 * 16), kAppendThreads, stream, attr);
  return launch_kernel(cfg, append_kernel, p);
}

cudaError_t launch_copy(const CopyParams& p, int sms, cudaStream_t stream) {
  constexpr int kRun = kCopyThreads * kCopyUnroll;
  const long long copies = static_cast<long long>(p.n) * p.pools.count * ((p.pools.pieces + kRun - 1) / kRun), most = 4ll * sms;
  const long long entries = p.job.renamed != nullptr ? static_cast<long long>(p.job.tables.sequences) * p.job.tables.cols : 0;
  const long long renames = (entries + kCopyThreads - 1) / kCopyThreads, total = copies > renames ? copies : renames;
  cudaLaunchAttribute attr[1];
  return launch_kernel(config(static_cast<unsigned>(total < most ? total : most), kCopyThreads, stream, attr), copy_kernel, p);
}

cudaError_t launch_free(const Tables& t, const int* sequences, int n, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  return launch_kernel(config(static_cast<unsigned>(n), 256, stream, attr), free_kernel, t, sequences, n);
}

cudaError_t launch_reserve(const Tables& t, const int* counts, int* scratch, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  return launch_kernel(config(1, kTableThreads, stream, attr), reserve_kernel, t, counts, scratch);
}

cudaError_t launch_fork(const Tables& t, const int* parents, const int* children, int n, int* source, int* target, int* list, int* count,
                        cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  return launch_kernel(config(1, kTableThreads, stream, attr), fork_pages_kernel, t, parents, children, n, source, target, list, count);
}

cudaError_t launch_compact(const Tables& t, int* new_references, int* renamed, int* source, int* target, int* count, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  return launch_kernel(config(1, kTableThreads, stream, attr), compact_pages_kernel, static_cast<const int*>(t.references), t.pages, new_references,
                       renamed, source, target, count);
}

}  // namespace cache
}  // namespace ditto_b200
