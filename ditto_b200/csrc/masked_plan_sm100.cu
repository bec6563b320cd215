// What stands around the kernels of the masked attention operators: which blocks the documents of a tile reach, the sum of the parts of
// items that several CTAs share, and the launches.
#include "masked_plan_sm100.cuh"

#include <climits>

#include "host_util.cuh"
#include "mlp_common.cuh"
#include "sm100_ptx.cuh"

namespace ditto_b200 {
namespace masked {
namespace {

constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int warp_min(int v) { return __reduce_min_sync(0xffffffffu, v); }
__device__ __forceinline__ int warp_max(int v) { return __reduce_max_sync(0xffffffffu, v); }

// Maximum over the threads up to this one; *before: of those in front of it (`none` for the first), *all: of all.
__device__ __forceinline__ int block_max(int v, int none, int* scratch, int* before, int* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl = max(incl, x);
  }
  const int left = __shfl_up_sync(0xffffffffu, incl, 1);
  __syncthreads();
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  static_assert(kPlanThreads == 1024, "a warp's value a lane");
  const int of_warp = scratch[lane], whole = max(none, warp_max(of_warp)), front = max(none, warp_max(lane < warp ? of_warp : INT_MIN));
  *before = lane == 0 ? front : max(front, left);
  *all = whole;
  return max(front, incl);
}

// One CTA a batch row.  Document ids may come in any order: a block is skipped where the ranges of ids of its keys and of a tile's queries
// do not meet, which for documents that follow one another are the blocks that hold none of the tile's, and never one that does.  Bound by the
// latency of its scans and of the reads between them: 10 us for four rows of 4096.
__global__ void __launch_bounds__(kPlanThreads, 1) document_plan_kernel(const int* documents, const int* prefix, int M, int L, int causal,
                                                                        int tile_tokens, int tiles, int2* runs, int* mixed,
                                                                        KeyBlock* key_blocks, int2* hulls, int2* key_hulls) {
  __shared__ int scratch[kPlanThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = kPlanThreads / 32;
  const int blocks = (L + kKeys - 1) / kKeys;
  const int* ids = documents + static_cast<size_t>(b) * L;
  KeyBlock* mine = key_blocks + static_cast<size_t>(b) * blocks;
  const int pre = prefix != nullptr ? prefix[b] : 0;
  // Runs of equal ids: a position's run begins at the last change of id up to it and ends at the first one behind it.  They are its document
  // where every id has one run, which is certain where the ids rise.
  int2* my_runs = runs + static_cast<size_t>(b) * L;
  constexpr int kEach = 4;                             // positions of a thread, one behind the other
  int begin = 0, highest = -1;
  bool falls = false;
  for (int base = 0; base < L; base += kPlanThreads * kEach) {
    const int k0 = base + static_cast<int>(threadIdx.x) * kEach;
    int last = k0 > 0 && k0 <= L ? ids[k0 - 1] : -1, change[kEach], id[kEach], latest = 0, most = -1, before, all;
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int k = k0 + u;
      id[u] = k < L ? ids[k] : -1;
      change[u] = k < L && (k == 0 || id[u] != last);
      if (change[u]) latest = k;
      last = id[u];
      most = max(most, id[u]);
    }
    block_max(latest, 0, scratch, &before, &all);
    int at = max(begin, before);
    begin = max(begin, all);
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      if (change[u]) at = k0 + u;
      if (k0 + u < L) my_runs[k0 + u].x = at;
    }
    block_max(most, -1, scratch, &before, &all);
    int up_to = max(highest, before);
    highest = max(highest, all);
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      falls |= change[u] && id[u] >= 0 && id[u] <= up_to;
      up_to = max(up_to, id[u]);
    }
  }
  const bool any_order = __syncthreads_or(falls);
  if (threadIdx.x == 0) mixed[b] = any_order;
  int end = 0;                                         // (of the positions counted from the row's end)
  for (int base = 0; base < L; base += kPlanThreads * kEach) {
    const int r0 = base + static_cast<int>(threadIdx.x) * kEach;
    int last = r0 > 0 && r0 <= L ? ids[L - r0] : -1, change[kEach], id[kEach], latest = 0, before, all;
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int r = r0 + u;
      id[u] = r < L ? ids[L - 1 - r] : -1;
      change[u] = r < L && (r == 0 || id[u] != last);
      if (change[u]) latest = r;
      last = id[u];
    }
    block_max(latest, 0, scratch, &before, &all);
    int at = max(end, before);
    end = max(end, all);
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int r = r0 + u, k = L - 1 - r;
      if (change[u]) at = r;
      if (r < L) my_runs[k] = id[u] < 0 ? make_int2(0, 0) : any_order ? make_int2(0, L) : make_int2(my_runs[k].x, L - at);
    }
  }
  for (int j = warp; j < blocks; j += warps) {
    int least = INT_MAX, most = -1;
#pragma unroll
    for (int u = 0; u < kKeys / 32; ++u) {
      const int k = j * kKeys + u * 32 + lane;
      if (k < L) {
        const int id = ids[k];
        if (id >= 0) least = min(least, id), most = max(most, id);
      }
    }
    least = warp_min(least), most = warp_max(most);
    if (lane == 0) mine[j] = {least, most};
  }
  __syncthreads();
  for (int tile = warp; tile < tiles; tile += warps) {
    const int first = tile * tile_tokens + L - M, last = min((tile + 1) * tile_tokens, M) - 1 + L - M;
    int least = INT_MAX, most = -1;
    for (int k = first + lane; k <= last; k += 32) {
      const int id = ids[k];
      if (id >= 0) least = min(least, id), most = max(most, id);
    }
    least = warp_min(least), most = warp_max(most);
    const int end = (visible_keys(last, L, causal, pre) + kKeys - 1) / kKeys;
    int lo = INT_MAX, hi = 0;
    for (int j = lane; j < end; j += 32) {
      const KeyBlock k = mine[j];
      if (k.least <= most && least <= k.most) lo = min(lo, j), hi = max(hi, j + 1);
    }
    lo = warp_min(lo), hi = warp_max(hi);
    if (lane == 0) hulls[static_cast<size_t>(b) * tiles + tile] = hi > 0 ? make_int2(lo, hi) : make_int2(0, 0);
  }
  if (key_hulls == nullptr) return;
  __syncthreads();
  // the other way round, for the gradients of a block of keys: the tiles whose hull holds it
  const int2* tile_hulls = hulls + static_cast<size_t>(b) * tiles;
  for (int j = warp; j < blocks; j += warps) {
    int lo = INT_MAX, hi = 0;
    for (int tile = lane; tile < tiles; tile += 32) {
      const int2 h = tile_hulls[tile];
      if (j >= h.x && j < h.y) lo = min(lo, tile), hi = max(hi, tile + 1);
    }
    lo = warp_min(lo), hi = warp_max(hi);
    if (lane == 0) key_hulls[static_cast<size_t>(b) * blocks + j] = hi > 0 ? make_int2(lo, hi) : make_int2(0, 0);
  }
}

// Sum of an item's parts, in the order of its keys: O = sum_p 2^(c (m_p - m)) O_p / sum_p 2^(c (m_p - m)) l_p.  CTAs (x, ..) for the item that
// CTA x of the forward kernel began, a warp a row.  Bound by reading the parts, which are in L2: 19 us for a chunk of 8192 tokens of 16 heads
// (37 MB), 5 us for 64 single tokens.
constexpr int kSumThreads = 256, kSumSlices = 16;
template <int D, bool BF16>
__global__ void __launch_bounds__(kSumThreads) sum_parts_kernel(const __grid_constant__ Params p, const int rows) {
  grid_dependency_wait();
  grid_launch_dependents();
  const PartDesc part = p.parts[blockIdx.x];
  if (part.last_cta < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = (part.last_cta - static_cast<int>(blockIdx.x)) / p.lanes + 1;
  Sequence q;
  q.load(p, part.seq);
  for (int r = blockIdx.y + kSumSlices * warp; r < rows; r += kSumSlices * (kSumThreads / 32)) {
    const int in_tile = r % kRows, token = part.first_token + (r / kRows) * p.tile_tokens + in_tile / p.group;
    if (in_tile / p.group >= p.tile_tokens || token >= q.tokens) continue;
    auto at = [&](int i) { return (static_cast<size_t>(blockIdx.x + i * p.lanes) * 2 + (i == 0 ? 1 : 0)) * rows + r; };
    float m = -INFINITY;
    for (int i = lane; i < n; i += 32) m = fmaxf(m, p.part_ml[at(i)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float total = 0.f, acc[D / 32];
#pragma unroll
    for (int u = 0; u < D / 32; ++u) acc[u] = 0.f;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float2 ml = p.part_ml[at(i)];
      const float* o = p.part_o + at(i) * D + lane * (D / 32);
      float v[D / 32];
      if constexpr (D == 128) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(o);
      else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(o);
      if (ml.y == 0.f) continue;                   // saw no key: its accumulator was not written
      const float f = ml.x == m ? 1.0f : ex2_approx((ml.x - m) * p.c);
      total = fmaf(f, ml.y, total);
#pragma unroll
      for (int u = 0; u < D / 32; ++u) acc[u] = fmaf(f, v[u], acc[u]);
    }
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    const int head = part.kv_head * p.group + in_tile % p.group, col = lane * (D / 32);
    if (col < p.d) {
      uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) +
                     2 * ((q.row0 + static_cast<long long>(token)) * p.out_token + head * p.out_head + col);
      if constexpr (D == 128) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv));
      } else {
        *reinterpret_cast<uint32_t*>(dst) = pack2<BF16>(acc[0] * inv, acc[1] * inv);
      }
    }
  }
}

cudaLaunchConfig_t config(int grid, int threads, cudaStream_t stream, cudaLaunchAttribute* attr, int slices = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), static_cast<unsigned>(slices), 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

}  // namespace

cudaError_t launch_document_plan(const int* documents, const int* prefix, int batch, int M, int L, int causal, int tile_tokens, int tiles,
                                 int2* runs, int* mixed, KeyBlock* key_blocks, int2* hulls, int2* key_hulls, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = config(batch, kPlanThreads, stream, attr);
  return launch_kernel(cfg, document_plan_kernel, documents, prefix, M, L, causal, tile_tokens, tiles, runs, mixed, key_blocks, hulls,
                       key_hulls);
}

cudaError_t launch_sum_parts(const Params& p, int d, bool bf16, int tiles, int grid, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = config(grid, kSumThreads, stream, attr, kSumSlices);
  const int rows = tiles == 0 ? 32 : tiles * kRows;
  if (d == 128) return bf16 ? launch_kernel(cfg, sum_parts_kernel<128, true>, p, rows) : launch_kernel(cfg, sum_parts_kernel<128, false>, p, rows);
  return bf16 ? launch_kernel(cfg, sum_parts_kernel<64, true>, p, rows) : launch_kernel(cfg, sum_parts_kernel<64, false>, p, rows);
}

cudaError_t launch_forward_any(const Params& p, int d, bool bf16, bool paged, int tiles, int grid, cudaStream_t stream) {
  if (paged) {
    if (d == 128) return bf16 ? launch_forward<128, true, true>(p, tiles, grid, stream) : launch_forward<128, false, true>(p, tiles, grid, stream);
    return bf16 ? launch_forward<64, true, true>(p, tiles, grid, stream) : launch_forward<64, false, true>(p, tiles, grid, stream);
  }
  if (d == 128) return bf16 ? launch_forward<128, true, false>(p, tiles, grid, stream) : launch_forward<128, false, false>(p, tiles, grid, stream);
  return bf16 ? launch_forward<64, true, false>(p, tiles, grid, stream) : launch_forward<64, false, false>(p, tiles, grid, stream);
}

}  // namespace masked
}  // namespace ditto_b200
