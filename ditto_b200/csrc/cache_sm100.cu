// Kernels of the paged key/value cache: appending, and the page operations.
#include "cache_sm100.cuh"

#include "host_util.cuh"
#include "masked_sm100.cuh"
#include "sm100_ptx.cuh"

namespace ditto_b200 {
namespace cache {
namespace {

constexpr int kAppendThreads = 256;

// A thread a 16-byte piece of a key row and of the value row beside it.  Bound by the bytes: each is read once and written once.
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

}  // namespace cache
}  // namespace ditto_b200
