// Gradients of masked attention, from P = 2^(c s - lse):  dV = P^T dO,  dS = P (dO V^T - delta) (1 - tanh^2),  dQ = scale dS K,
// dK = scale dS^T Q,  delta_i = sum_d dO_id O_id.
//
// Four launches: delta with the other things the kernels need of a query row, in tile order; the queries' gradients; the keys'; the sum of
// what several CTAs have of a block of keys.  The two in the middle compute the scores and dO V^T each for themselves, and the queries' one P K
// as well (eight products instead of five), so that every sum stays in tensor memory in one CTA, in a fixed order: no atomics, no
// accumulator that passes through memory for every block, the same bits every time.
//
// Sixteen warps of arithmetic, four threads a row with 32 columns each, two MMA warps and a producer.  Tiles come in halves of 64 rows or
// keys through a ring of four: a half's loads go out as soon as the half two before is done with.
// Queries: a tile stays, the blocks of keys pass; P and dS go over the scores and dP, the first operands of P K and dS K.  delta is set right
// from sum_j P (dP - delta), see there.
// Keys: a block of 128 keys stays, the query tiles pass.  S^T = K Q^T and dP^T = V dO^T have keys as rows, so that P^T and dS^T go back to
// tensor memory as the first operands of dV += P^T dO and dK += dS^T Q without a transposition.  The tiles of all blocks are dealt out in
// equal shares to the CTAs (causal masks make blocks unequal, shared key heads make them few and long); blocks that a share cuts are
// summed from fp32 parts, in order.
//
// What bounds it: the tensor pipe, at eight products, beside the arithmetic.  16 heads, 8192 x 8192, bf16: d = 128 full 1674 us (821 TFLOP/s
// counted at five products, 1310 at eight), causal 957 us; d = 64 causal 804 us (the products' shapes are half as deep, the arithmetic is the
// same).  Of 935 us with a bias by distance, fp16: rows 26, queries 380, keys 487, sums 11 us.
//
// fp16: P is taken times 2^14 and dS times a power of two from the largest row norms of dO and V, so that neither leaves the type's range
// nor falls below its normal numbers as weights of a few thousand keys would.
#include <atomic>
#include <climits>

#include "host_util.cuh"
#include "masked_backward_sm100.cuh"
#include "mlp_common.cuh"
#include "sm100_ptx.cuh"
#include "softmax_step.cuh"

#ifndef DITTO_MASKED_BACKWARD_PART
#define DITTO_MASKED_BACKWARD_PART 0
#endif

namespace ditto_b200 {
namespace masked {
namespace {

constexpr int kComputeWarps = 16, kThreads = 32 * (kComputeWarps + 3);
constexpr int kProducerWarp = kComputeWarps, kMmaWarp = kComputeWarps + 1;      // (two MMA warps)
constexpr uint32_t kTmemCols = 512, kColS = 0, kColDp = 128, kColAcc = 256;
constexpr int kSegs = 4;
constexpr int kCols = 32;                              // columns of a score tile that one of a row's four threads has
constexpr float kPScaleLog2 = 14.0f;                   // of P in fp16

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// 2^k and 2^-k for dS in fp16: |dS| <= |dO_i| (|V_j| + |O_i|) <= 2 max |dO| max |V|, which 2^k takes to at most 2^15.
template <bool BF16>
__device__ __forceinline__ void ds_scale(const BackwardParams& p, float* up, float* down) {
  *up = *down = 1.0f;
  if constexpr (!BF16) {
    const float a = __uint_as_float(p.norms[0]), b = __uint_as_float(p.norms[1]);      // squares
    const float bound = sqrtf(a) * sqrtf(b);
    if (bound > 0.f && bound < INFINITY) {
      const int e = min(100, max(-100, 14 - (static_cast<int>(__float_as_uint(bound) >> 23) - 127 + 1)));
      *up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      *down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    }
  }
}

// ------------------------------------------------------------------ rows
constexpr int kRowThreads = 128;

template <bool BF16>
__device__ __forceinline__ void dot8(uint4 a, uint4 b, float& dot, float& norm_a) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = unpack2<BF16>(x[i]), v = unpack2<BF16>(y[i]);
    dot = fmaf(u.x, v.x, fmaf(u.y, v.y, dot));
    norm_a = fmaf(u.x, u.x, fmaf(u.y, u.y, norm_a));
  }
}

// A CTA half a tile at a time, LANES threads a row of it and kRowsAtOnce rows in flight a thread.  Bound by reading out and its gradient once:
// 67 MB of them in 26 us (16 heads of 128, 8192 tokens, fp16, with the values for their norms), 34 MB in 12 us (2 x 2047, bf16).
template <bool BF16, int LANES>
__global__ void __launch_bounds__(kRowThreads) backward_rows_kernel(const __grid_constant__ BackwardParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  constexpr int kSpan = kRowThreads / LANES, kRowsAtOnce = kHalf / kSpan;
  const int lane = threadIdx.x % LANES, first = threadIdx.x / LANES, pieces = p.d / 8;
  const int halves = p.items * 2;
  float norm_g = 0.f, norm_v = 0.f;
  for (int at = blockIdx.x; at < halves; at += gridDim.x) {
    const int g = at & 1, tile = at / 2 % p.tiles, kv_head = at / 2 / p.tiles % p.kv_heads, b = at / 2 / p.tiles / p.kv_heads;
    const int token0 = tile * p.tile_tokens + g * p.half_tokens;
    uint4 vg[kRowsAtOnce], vo[kRowsAtOnce];
    int token[kRowsAtOnce], head[kRowsAtOnce], doc[kRowsAtOnce];
    float lse[kRowsAtOnce], slope[kRowsAtOnce];
    bool valid[kRowsAtOnce];
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int r = first + i * kSpan, of_half = r / p.half_heads, in_group = g * p.head_step + r - of_half * p.half_heads;
      token[i] = token0 + of_half;
      head[i] = kv_head * p.group + in_group;
      valid[i] = r < p.half_rows && in_group < p.group && token[i] < p.M;
      vg[i] = vo[i] = make_uint4(0, 0, 0, 0);
      lse[i] = -INFINITY, doc[i] = -1, slope[i] = 0.f;
      if (valid[i] && lane == 0) {                     // (all loads of a round go out together)
        lse[i] = p.lse[(static_cast<size_t>(b) * p.M + token[i]) * p.heads + head[i]];
        if (p.documents != nullptr) doc[i] = p.documents[static_cast<size_t>(b) * p.L + token[i] + p.L - p.M];
        if (p.slopes != nullptr) slope[i] = p.slopes[head[i]] * -1.4426950408889634f;
      }
      if (valid[i] && lane < pieces) {
        vg[i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.grad) + 2 * (b * p.g_stride[0] + token[i] * p.g_stride[1] + head[i] * p.g_stride[2]) + lane * 16);
        vo[i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.o) + 2 * (b * p.o_stride[0] + token[i] * p.o_stride[1] + head[i] * p.o_stride[2]) + lane * 16);
      }
    }
    HalfRows& t = p.rows[at];
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      float dot = 0.f, norm = 0.f;
      dot8<BF16>(vg[i], vo[i], dot, norm);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) {
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (!BF16) norm += __shfl_xor_sync(0xffffffffu, norm, o);
      }
      norm_g = fmaxf(norm_g, norm);
      if (lane == 0) {
        const int r = first + i * kSpan, pos = token[i] + p.L - p.M;
        t.lse[r] = lse[i] == -INFINITY ? -INFINITY : fmaf(lse[i], -1.4426950408889634f, BF16 ? 0.f : kPScaleLog2);
        t.delta[r] = -dot;
        t.doc[r] = doc[i];
        t.slope[r] = slope[i];
        t.pos[r] = static_cast<float>(pos);
      }
    }
  }
  if constexpr (!BF16) {
    // (the loop's bounds are those of whole warps: shuffles)
    constexpr int kPerWarp = 32 / LANES;
    const long long keys = static_cast<long long>(p.batch) * p.L * p.kv_heads, step = static_cast<long long>(gridDim.x) * kSpan;
    for (long long at = static_cast<long long>(blockIdx.x) * kSpan + first; at - first % kPerWarp < keys; at += step) {
      const long long of_head = at / p.kv_heads;
      const int h = static_cast<int>(at - of_head * p.kv_heads), b = static_cast<int>(of_head / p.L), j = static_cast<int>(of_head - static_cast<long long>(b) * p.L);
      float dot = 0.f, norm = 0.f;
      if (at < keys && lane < pieces) {
        const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.v) + 2 * (b * p.v_stride[0] + j * p.v_stride[1] + h * p.v_stride[2]) + lane * 16);
        dot8<BF16>(v, v, dot, norm);
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) norm += __shfl_xor_sync(0xffffffffu, norm, o);
      norm_v = fmaxf(norm_v, norm);
    }
    // the largest of all: the order of atomics does not show in it
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      norm_g = fmaxf(norm_g, __shfl_xor_sync(0xffffffffu, norm_g, o));
      norm_v = fmaxf(norm_v, __shfl_xor_sync(0xffffffffu, norm_v, o));
    }
    if ((threadIdx.x & 31) == 0) {
      atomicMax(p.norms, __float_as_uint(norm_g));
      atomicMax(p.norms + 1, __float_as_uint(norm_v));
    }
  }
}

struct KeySegment {
  int item, seq, kv_head, block;
  int lo, hi;               // query tiles
  int prefix, part, units, at_unit, tile0, valid;
};

template <int D>
struct Layout {
  static constexpr int kAtoms = D / 64, kTile = 128 * D * 2;
  static constexpr int kOffA = 0, kOffB = kTile;                 // what stays: K and V, or Q and dO
  static constexpr int kHalfTile = kTile / 2;
  static constexpr int kOffRing = 2 * kTile;                     // four stages of what passes: halves of Q and dO, or of K and V
  static constexpr int kOffRows = kOffRing + 4 * kTile;          // [4] HalfRows
  static constexpr int kOffBar = kOffRows + 4 * static_cast<int>(sizeof(HalfRows));
  static constexpr int kOffSeg = kOffBar + 512;
  static constexpr int kBytes = kOffSeg + 512 + 1024;
};

struct Bars {
  uint64_t keep_full, keep_empty;
  uint64_t full[4], empty[4];
  uint64_t s_full[2], p_full[2], dp_full[2], ds_full[2], acc_done, acc_free, sums_full;
  uint64_t seg_full[kSegs], seg_empty[kSegs];
  uint32_t tmem_base, abort_word;
  int start_item, start_tile, left, per_cta;
  int scan[kThreads / 32 + 1];
};
static_assert(sizeof(Bars) <= 512, "barrier block too large");

// Query tiles [x, y) that see block j of the keys of batch entry b.
__device__ __forceinline__ int2 tiles_of_block(const BackwardParams& p, int b, int j) {
  if (p.documents != nullptr) return p.key_hulls[static_cast<size_t>(b) * p.blocks + j];
  int first = 0;
  if (p.causal && !(p.prefix != nullptr && p.prefix[b] > j * kKeys)) first = max(0, j * kKeys - (p.L - p.M));
  return first < p.M ? make_int2(first / p.tile_tokens, p.tiles) : make_int2(0, 0);
}
__device__ __forceinline__ int units_of_item(const BackwardParams& p, int item) {
  const int j = item % p.blocks, b = item / p.blocks / p.kv_heads;
  const int2 t = tiles_of_block(p, b, j);
  return max(1, t.y - t.x);          // (blocks that nobody sees get their zeros)
}

// The share of this CTA: the tiles of all blocks, in order, in gridDim.x equal shares.
__device__ __forceinline__ void find_share(const BackwardParams& p, Bars* bar) {
  constexpr int kWarps = kThreads / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, items = p.batch * p.kv_heads * p.blocks;
  int sum = 0;
  for (int i = tid; i < items; i += kThreads) sum += units_of_item(p, i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) bar->scan[warp] = sum;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < kWarps; ++w) total += bar->scan[w];
  const int grid = gridDim.x, per = max(1, (total + grid - 1) / grid);
  const int u0 = static_cast<int>(min(static_cast<long long>(per) * blockIdx.x, static_cast<long long>(total))), left = min(per, total - u0);
  if (tid == 0) bar->left = 0, bar->per_cta = per, bar->start_item = 0, bar->start_tile = 0;
  int before = 0;
  for (int base = 0; base < items && before <= u0; base += kThreads) {
    const int cost = base + tid < items ? units_of_item(p, base + tid) : 0;
    int incl = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) bar->scan[warp] = incl;
    __syncthreads();
    int offset = before, all = before;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) offset += bar->scan[w];
      all += bar->scan[w];
    }
    const int at = u0 - (offset + incl - cost);
    if (left > 0 && at >= 0 && at < cost) bar->start_item = base + tid, bar->start_tile = at, bar->left = left;
    before = all;
  }
  __syncthreads();
}

// Rows of a half that the loads do not write (a group that does not divide 64): as rows of the sums they have to be zeros.
__device__ __forceinline__ void zero_unused_rows(uint8_t* half, int atoms, int from) {
  for (int a = 0; a < atoms; ++a)
    for (int i = from * 8 + static_cast<int>(threadIdx.x); i < kHalf * 8; i += kThreads)
      *reinterpret_cast<uint4*>(half + a * (kHalf * 128) + i * 16) = make_uint4(0, 0, 0, 0);
}

// 128 rows of keys, or of queries (`heads` apart from the one that tokens step by), in two boxes of 64.
template <int D>
__device__ __forceinline__ void load_halves(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int x1, int x1_step, int x2, int x2_step, int x3) {
  for (int a = 0; a < D / 64; ++a)
    for (int g = 0; g < 2; ++g) tma_load_4d(dst + a * (kRows * 128) + g * (kHalf * 128), map, bar, a * 64, x1 + g * x1_step, x2 + g * x2_step, x3);
}

// What the two MMA warps of either kernel do (a converged warp, an elected lane issues).  Warp 0: scores S of what stays at kOffA with the
// first operand of a stage, and the first sum, from P; warp 1: dP of what stays at kOffB with the second operand, and the second sum, from dS.
// Both sums' other operand is an operand of the stage too, its rows as the reduction: `sum_of` says which, 0 or 1.  What
// stays has 128 rows, a stage holds half of the 128 that pass: the halves have score columns of their own, so that one's products run
// under the other's arithmetic.  `range` gives the tiles or blocks of a segment.
template <int D, bool BF16, class Seg, class Range>
__device__ __forceinline__ void issue_products(uint8_t* smem, Bars* bar, uint32_t tmem_base, const Seg* segments, int which, int lane, int sum_of,
                                               Range range) {
  using LO = Layout<D>;
  constexpr int kTile = LO::kTile, kHalfTile = LO::kHalfTile;
  volatile uint32_t* abort_word = &bar->abort_word;
  const uint32_t issuer = elect_one();
  const uint32_t idesc_s = umma_idesc_f16(BF16, kRows, kHalf, false, false);
  const uint32_t idesc_acc = umma_idesc_f16(BF16, kRows, D, false, true);
  const uint64_t da = umma_desc_sw128(smem_u32(smem + (which == 0 ? LO::kOffA : LO::kOffB)), 16, 1024);
  const uint64_t db0 = umma_desc_sw128(smem_u32(smem + LO::kOffRing + which * kHalfTile), 16, 1024);
  const uint64_t dr0 = umma_desc_sw128(smem_u32(smem + LO::kOffRing + sum_of * kHalfTile), kHalf * 128, 1024);
  const uint32_t d_first = tmem_base + (which == 0 ? kColS : kColDp), d_acc = tmem_base + kColAcc + which * D;
  uint64_t* first_full = which == 0 ? bar->s_full : bar->dp_full;
  uint64_t* back_full = which == 0 ? bar->p_full : bar->ds_full;
  auto wait = [&](uint64_t* b, uint32_t parity, uint32_t code) {
    const bool r = __all_sync(0xffffffffu, mbar_wait(b, parity, abort_word, code));
    tc_fence_after_sync();
    return r;
  };
  // the scores of half g of tile or block n: stage 2 n + g of the ring
  auto issue_first = [&](int n, int g) {
    const uint64_t db = db0 + ((((2 * n + g) & 3) * kTile) >> 4);
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      umma_ss_elected(d_first + g * kHalf, da + (((i / 4) * (kRows * 128) + (i % 4) * 32) >> 4), db + (((i / 4) * (kHalf * 128) + (i % 4) * 32) >> 4),
                      idesc_s, i > 0 ? 1u : 0u, issuer);
    umma_commit_elected(&first_full[g], issuer);
  };
  auto wait_half = [&](int n, int g) { return wait(&bar->full[(2 * n + g) & 3], (n >> 1) & 1, 0x310 + g); };
  uint32_t keeps = 0;
  int n = 0;
  bool ok = true;
  for (int segs = 0; ok; ++segs) {
    const int slot = segs % kSegs;
    ok = wait(&bar->seg_full[slot], (segs / kSegs) & 1, 0x350);
    if (!ok || !segments[slot].valid) break;
    int lo, hi;
    range(segments[slot], &lo, &hi);
    mbar_arrive_warp(&bar->seg_empty[slot], lane);
    if (lo >= hi) continue;
    if (!(ok = wait(&bar->keep_full, keeps & 1, 0x300) && wait_half(n, 0))) break;
    issue_first(n, 0);
    if (!(ok = wait_half(n, 1))) break;
    issue_first(n, 1);
    for (int i = lo; i < hi; ++i, ++n) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint64_t dr = dr0 + ((((2 * n + g) & 3) * kTile) >> 4);
        if (i + 1 < hi && !(ok = ok && wait_half(n + 1, g))) break;      // (there long before its turn)
        if (!(ok = ok && wait(&back_full[g], n & 1, 0x340 + which))) break;
        if (g == 0 && i == lo && !(ok = wait(&bar->acc_free, (keeps & 1) ^ 1, 0x320))) break;      // (at once the first time)
#pragma unroll
        for (int q = 0; q < kHalf / 16; ++q)
          umma_ts_elected(d_acc, d_first + g * kHalf + (q / 2) * kCols + (q % 2) * 8, dr + ((q * 2048) >> 4), idesc_acc,
                          g > 0 || q > 0 || i > lo ? 1u : 0u, issuer);
        umma_commit_elected(&bar->empty[(2 * n + g) & 3], issuer);
        if (i + 1 < hi) issue_first(n + 1, g);
      }
      if (!ok) break;
    }
    if (!ok) break;
    umma_commit_elected(&bar->keep_empty, issuer);
    umma_commit_elected(&bar->acc_done, issuer);
    ++keeps;
  }
}

}  // namespace

// ------------------------------------------------------------------ gradients of keys and values
template <int D, bool BF16, bool CAPPED, bool BIASED>
__global__ void __launch_bounds__(kThreads, 1) backward_keys_kernel(const __grid_constant__ BackwardParams p) {
  using LO = Layout<D>;
  constexpr int kAtoms = LO::kAtoms, kTile = LO::kTile, kHalfTile = LO::kHalfTile;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bar = reinterpret_cast<Bars*>(smem + LO::kOffBar);
  KeySegment* segments = reinterpret_cast<KeySegment*>(smem + LO::kOffSeg);
  static_assert(sizeof(KeySegment) * kSegs <= 512, "segments");
  volatile uint32_t* abort_word = &bar->abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bar->keep_full, 1);
    mbar_init(&bar->keep_empty, 2);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 2);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&bar->s_full[g], 1);
      mbar_init(&bar->p_full[g], kComputeWarps / 2);
      mbar_init(&bar->dp_full[g], 1);
      mbar_init(&bar->ds_full[g], kComputeWarps / 2);
    }
    mbar_init(&bar->acc_done, 2);
    mbar_init(&bar->acc_free, kComputeWarps);
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(&bar->seg_full[i], 1);
      mbar_init(&bar->seg_empty[i], kComputeWarps + 2);
    }
    bar->abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&bar->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  if (p.half_rows < kHalf) {
    for (int i = 0; i < 8; ++i) zero_unused_rows(smem + LO::kOffRing + i * kHalfTile, kAtoms, p.half_rows);
    fence_proxy_async_smem();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = bar->tmem_base;
  grid_dependency_wait();
  grid_launch_dependents();
  find_share(p, bar);

  if (warp == kProducerWarp) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const uint32_t half_bytes = static_cast<uint32_t>(p.half_rows) * 128 * kAtoms;
      int item = bar->start_item, skip = bar->start_tile, left = bar->left, done = 0, n = 0, keeps = 0;
      bool ok = true;
      for (int segs = 0; ok; ++segs) {
        const int slot = segs % kSegs;
        ok = mbar_wait(&bar->seg_empty[slot], ((segs / kSegs) & 1) ^ 1, abort_word, 0x120);
        if (!ok) break;
        KeySegment s;
        s.valid = left > 0;
        if (s.valid) {
          s.item = item;
          s.block = item % p.blocks;
          s.kv_head = item / p.blocks % p.kv_heads;
          s.seq = item / p.blocks / p.kv_heads;
          const int2 t = tiles_of_block(p, s.seq, s.block);
          s.units = max(1, t.y - t.x);
          const int take = min(left, s.units - skip);
          s.lo = t.x + skip;
          s.hi = min(t.y, t.x + skip + take);
          s.part = skip > 0 ? 0 : take < s.units ? 1 : -1;
          s.at_unit = done;
          s.prefix = p.prefix != nullptr ? p.prefix[s.seq] : 0;
          s.tile0 = n;
          left -= take;
          done += take;
          ++item;
          skip = 0;
        }
        segments[slot] = s;
        mbar_arrive(&bar->seg_full[slot]);
        if (!s.valid) break;
        if (s.lo >= s.hi) continue;
        ok = mbar_wait(&bar->keep_empty, (keeps & 1) ^ 1, abort_word, 0x100);
        if (!ok) break;
        ++keeps;
        mbar_arrive_expect_tx(&bar->keep_full, 2 * kTile);
        load_halves<D>(smem + LO::kOffA, &p.map_k, &bar->keep_full, s.block * kKeys, kHalf, s.kv_head, 0, s.seq);
        load_halves<D>(smem + LO::kOffB, &p.map_v, &bar->keep_full, s.block * kKeys, kHalf, s.kv_head, 0, s.seq);
        for (int i = s.lo; ok && i < s.hi; ++i, ++n) {
          for (int g = 0; g < 2; ++g) {
            const int h = 2 * n + g, st = h & 3;
            ok = mbar_wait(&bar->empty[st], ((h >> 2) & 1) ^ 1, abort_word, 0x110);
            if (!ok) break;
            mbar_arrive_expect_tx(&bar->full[st], 2 * half_bytes + static_cast<uint32_t>(sizeof(HalfRows)));
            uint8_t* dst = smem + LO::kOffRing + st * kTile;
            const int head = s.kv_head * p.group + g * p.head_step, token = i * p.tile_tokens + g * p.half_tokens;
            for (int a = 0; a < kAtoms; ++a) {
              tma_load_4d(dst + a * (kHalf * 128), &p.map_q, &bar->full[st], a * 64, head, token, s.seq);
              tma_load_4d(dst + kHalfTile + a * (kHalf * 128), &p.map_do, &bar->full[st], a * 64, head, token, s.seq);
            }
            bulk_load(smem + LO::kOffRows + st * sizeof(HalfRows), p.rows + ((static_cast<size_t>(s.seq) * p.kv_heads + s.kv_head) * p.tiles + i) * 2 + g,
                      sizeof(HalfRows), &bar->full[st]);
          }
        }
      }
    }
  } else if (warp >= kMmaWarp) {
    // ------------------------------------------------------------ MMA: warp 0 S^T = K Q^T and dV += P^T dO, warp 1 dP^T = V dO^T and dK += dS^T Q
    const int which = warp - kMmaWarp;
    issue_products<D, BF16>(smem, bar, tmem_base, segments, which, lane, which ^ 1, [](const KeySegment& s, int* lo, int* hi) { *lo = s.lo, *hi = s.hi; });
  } else {
    // ------------------------------------------------------------ arithmetic: thread a key and a quarter of the tile's rows; warps 0-7 the
    // first half of them, 8-15 the second, each half with buffers of its own
    const int quad = warp & 3, part_of_row = warp >> 2, g = warp >> 3, sub = part_of_row & 1, row = quad * 32 + lane;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t s_col = lane_base + kColS + part_of_row * kCols, dp_col = lane_base + kColDp + part_of_row * kCols;
    const float c = p.c;
    float up, down;
    ds_scale<BF16>(p, &up, &down);
    const float p_down = BF16 ? 1.0f : 1.0f / 16384.0f;
    const float f = BF16 ? 1.0f : up * p_down;
    int n = 0;
    uint32_t accs = 0;
    bool ok = true;
    if (threadIdx.x == 0) p.parts[blockIdx.x].last_cta = -1;
    for (int segs = 0;; ++segs) {
      const int slot = segs % kSegs;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar->seg_full[slot], (segs / kSegs) & 1, abort_word, 0x840));
      if (!ok) break;
      const KeySegment& s = segments[slot];
      if (!s.valid) break;
      const int lo = s.lo, hi = s.hi, key = s.block * kKeys + row;
      // positions that see the key: from `first` up to `end` (causal, and not in the prefix that all see; documents)
      int first = p.causal && !(key < s.prefix) ? key : INT_MIN / 256, end = INT_MAX / 256, doc = -2;
      bool mixed = false;
      if (p.documents != nullptr) {
        if (key < p.L) {
          const size_t at = static_cast<size_t>(s.seq) * p.L + key;
          const int2 run = p.runs[at];
          first = max(first, run.x);
          end = run.y;
          doc = p.documents[at];
        }
        mixed = p.mixed[s.seq] != 0;
      }
      const int first_of_all = __reduce_max_sync(0xffffffffu, first), end_of_all = __reduce_min_sync(0xffffffffu, end);
      for (int i = lo; i < hi; ++i, ++n) {
        const int st = (2 * n + g) & 3;
        const HalfRows& rows = *reinterpret_cast<const HalfRows*>(smem + LO::kOffRows + st * sizeof(HalfRows));
        ok = mbar_wait(&bar->full[st], (n >> 1) & 1, abort_word, 0x850);
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&bar->s_full[g], n & 1, abort_word, 0x800));
        if (!ok) break;
        tc_fence_after_sync();
        const int pos0 = p.L - p.M + i * p.tile_tokens + g * p.half_tokens;      // of the half's first row; columns from .. to - 1 see the key
        const bool cut = first_of_all > pos0, cut_end = end_of_all < pos0 + kHalf;      // (a half has at most that many tokens)
        float w[kCols] = {};
        {
          uint32_t sv[32];
          tmem_ld_x32_wait(s_col, sv);
          // (w holds what dS is the product of with dP - delta: first 1 - tanh^2, then that times the weight)
          if constexpr (CAPPED) {
              capped(sv, p.cap_in, 1.0f);
              const uint64_t one2 = pack_f32x2(1.0f, 1.0f), out2 = pack_f32x2(p.cap_out, p.cap_out);
#pragma unroll
              for (int u = 0; u < 32; u += 2) {
                const uint64_t t = pack_f32x2(__uint_as_float(sv[u]), __uint_as_float(sv[u + 1]));
                unpack_f32x2(fma_f32x2(mul_f32x2(t, pack_f32x2(-1.0f, -1.0f)), t, one2), w[u], w[u + 1]);
                float y0, y1;
                unpack_f32x2(mul_f32x2(t, out2), y0, y1);
                sv[u] = __float_as_uint(y0), sv[u + 1] = __float_as_uint(y1);
              }
          }
          if constexpr (BIASED) {
            if (p.slopes != nullptr) {
              const float sc = CAPPED ? 1.0f : p.score_log2, at = static_cast<float>(key);
              const uint64_t sc2 = pack_f32x2(sc, sc), at2 = pack_f32x2(-at, -at);
#pragma unroll
              for (int u = 0; u < 32; u += 4) {
                const float4 sl = *reinterpret_cast<const float4*>(&rows.slope[sub * kCols + u]);
                const float4 ps = *reinterpret_cast<const float4*>(&rows.pos[sub * kCols + u]);
#pragma unroll
                for (int q = 0; q < 4; q += 2) {
                  float d0, d1;
                  unpack_f32x2(add_f32x2(q == 0 ? pack_f32x2(ps.x, ps.y) : pack_f32x2(ps.z, ps.w), at2), d0, d1);
                  const uint64_t bias = mul_f32x2(q == 0 ? pack_f32x2(sl.x, sl.y) : pack_f32x2(sl.z, sl.w), pack_f32x2(fabsf(d0), fabsf(d1)));
                  float y0, y1;
                  unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(sv[u + q]), __uint_as_float(sv[u + q + 1])), sc2, bias), y0, y1);
                  sv[u + q] = __float_as_uint(y0), sv[u + q + 1] = __float_as_uint(y1);
                }
              }
            }
          }
          if (mixed) {
#pragma unroll
              for (int u = 0; u < 32; u += 4) {
                const int4 d = *reinterpret_cast<const int4*>(&rows.doc[sub * kCols + u]);
                if (d.x != doc) sv[u] = __float_as_uint(-INFINITY);
                if (d.y != doc) sv[u + 1] = __float_as_uint(-INFINITY);
                if (d.z != doc) sv[u + 2] = __float_as_uint(-INFINITY);
                if (d.w != doc) sv[u + 3] = __float_as_uint(-INFINITY);
              }
          }
          if (cut) {
            const int from = first > pos0 ? min(first - pos0, kHalf) * p.half_heads - sub * kCols : 0;
#pragma unroll
            for (int u = 0; u < 32; ++u)
              if (u < from) sv[u] = __float_as_uint(-INFINITY);
          }
          if (cut_end) {
            const int to = min(max(end - pos0, 0), kHalf) * p.half_heads - sub * kCols;
#pragma unroll
            for (int u = 0; u < 32; ++u)
              if (u >= to) sv[u] = __float_as_uint(-INFINITY);
          }
          const uint64_t c2 = pack_f32x2(c, c);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t pk[8];
#pragma unroll
            for (int v = 0; v < 8; v += 2) {
              const int u = q * 16 + v * 2;
              const float4 lse = *reinterpret_cast<const float4*>(&rows.lse[sub * kCols + u]);
              const uint64_t p01 = softmax_weights(sv[u], sv[u + 1], c2, pack_f32x2(lse.x, lse.y), false);
              const uint64_t p23 = softmax_weights(sv[u + 2], sv[u + 3], c2, pack_f32x2(lse.z, lse.w), false);
              float p0, p1, p2, p3;
              unpack_f32x2(p01, p0, p1);
              unpack_f32x2(p23, p2, p3);
              pk[v] = pack2<BF16>(p0, p1);
              pk[v + 1] = pack2<BF16>(p2, p3);
              uint64_t w01 = p01, w23 = p23;
              if constexpr (CAPPED) w01 = mul_f32x2(w01, pack_f32x2(w[u], w[u + 1])), w23 = mul_f32x2(w23, pack_f32x2(w[u + 2], w[u + 3]));
              if constexpr (!BF16) w01 = mul_f32x2(w01, pack_f32x2(f, f)), w23 = mul_f32x2(w23, pack_f32x2(f, f));
              unpack_f32x2(w01, w[u], w[u + 1]);
              unpack_f32x2(w23, w[u + 2], w[u + 3]);
            }
            // (packed weights go over the first half of this thread's own columns)
            tmem_st_x8(s_col + q * 8, pk);
          }
        }
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive_warp(&bar->p_full[g], lane);

        ok = __all_sync(0xffffffffu, mbar_wait(&bar->dp_full[g], n & 1, abort_word, 0x810));
        if (!ok) break;
        tc_fence_after_sync();
        {
          uint32_t dp[32];
          tmem_ld_x32_wait(dp_col, dp);
          uint32_t pk[16];
#pragma unroll
          for (int u = 0; u < 32; u += 4) {
            const float4 de = *reinterpret_cast<const float4*>(&rows.delta[sub * kCols + u]);
            auto product = [&](int i, float d0, float d1) {
              float x0, x1;
              unpack_f32x2(mul_f32x2(pack_f32x2(w[i], w[i + 1]), add_f32x2(pack_f32x2(__uint_as_float(dp[i]), __uint_as_float(dp[i + 1])), pack_f32x2(d0, d1))), x0, x1);
              return pack2<BF16>(x0, x1);
            };
            pk[u / 2] = product(u, de.x, de.y);
            pk[u / 2 + 1] = product(u + 2, de.z, de.w);
          }
          tmem_st_x16(dp_col, pk);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive_warp(&bar->ds_full[g], lane);
      }
      if (!ok) break;

      // the block's gradients, or this part of their sums: dV in the first D columns, dK behind them; a quarter of the columns a thread
      const bool has = lo < hi;
      if (has) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bar->acc_done, accs & 1, abort_word, 0x830));
        ++accs;
        if (!ok) break;
        tc_fence_after_sync();
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float scale = m == 0 ? p_down : p.scale * down;
        uint8_t* dst = static_cast<uint8_t*>(m == 0 ? p.dv : p.dk) + 2 * ((static_cast<size_t>(s.seq) * p.L + key) * p.kv_heads + s.kv_head) * p.d;
        float* part = p.part + (((static_cast<size_t>(blockIdx.x) * 2 + max(s.part, 0)) * 2 + m) * kKeys + row) * D;
#pragma unroll
        for (int cc = 0; cc < D / 4; cc += 16) {
          const int col = part_of_row * (D / 4) + cc;
          uint32_t x[16];
          if (has) {
            tmem_ld_x16_wait(lane_base + kColAcc + m * D + col, x);
          } else {
#pragma unroll
            for (int u = 0; u < 16; ++u) x[u] = 0u;
          }
          if (m == 1 && cc + 16 == D / 4) {
            tc_fence_before_sync();
            if (has) mbar_arrive_warp(&bar->acc_free, lane);
          }
          if (key >= p.L) continue;
          if (s.part >= 0) {
#pragma unroll
            for (int u = 0; u < 16; u += 4) *reinterpret_cast<uint4*>(part + col + u) = make_uint4(x[u], x[u + 1], x[u + 2], x[u + 3]);
            continue;
          }
#pragma unroll
          for (int u = 0; u < 16; u += 8) {
            uint32_t v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = pack2<BF16>(__uint_as_float(x[u + 2 * q]) * scale, __uint_as_float(x[u + 2 * q + 1]) * scale);
            if (col + u < p.d) *reinterpret_cast<uint4*>(dst + 2 * (col + u)) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      }
      if (s.part == 1 && threadIdx.x == 0) {
        const long long first_unit = static_cast<long long>(blockIdx.x) * bar->per_cta + s.at_unit;
        p.parts[blockIdx.x] = {s.item, static_cast<int>((first_unit + s.units - 1) / bar->per_cta)};
      }
      mbar_arrive_warp(&bar->seg_empty[slot], lane);
    }
  }

  if (bar->abort_word != 0u) {
    for (int t = 0; t < 64; ++t) __nanosleep(1000);      // loads in flight land before their shared memory is released
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tmem_dealloc(tmem_base, kTmemCols);
    if (lane == 0 && bar->abort_word != 0 && p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(bar->abort_word));
  }
}

namespace {

// Sums of the parts of a block that several CTAs had, in the order of its tiles.  CTAs (x, ..) for the block that CTA x of the kernel above
// began, kSumSlices of them with 1 / kSumSlices of its values each.  Bound by reading the parts: 11 us for 148 CTAs' with heads of 128.
constexpr int kSumThreads = 256, kSumSlices = 8;
template <int D, bool BF16>
__global__ void __launch_bounds__(kSumThreads) sum_key_parts_kernel(const __grid_constant__ BackwardParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const KeyPartDesc part = p.parts[blockIdx.x];
  if (part.last_cta < 0) return;
  const int block = part.item % p.blocks, kv_head = part.item / p.blocks % p.kv_heads, seq = part.item / p.blocks / p.kv_heads;
  float up, down;
  ds_scale<BF16>(p, &up, &down);
  for (int i = blockIdx.y * kSumThreads + threadIdx.x; i < 2 * kKeys * (D / 8); i += kSumThreads * kSumSlices) {
    const int col = i % (D / 8) * 8, row = i / (D / 8) % kKeys, m = i / (D / 8) / kKeys, key = block * kKeys + row;
    if (key >= p.L || col >= p.d) continue;
    float x[8] = {};
    for (int cta = blockIdx.x; cta <= part.last_cta; ++cta) {
      const float* src = p.part + (((static_cast<size_t>(cta) * 2 + (cta == static_cast<int>(blockIdx.x) ? 1 : 0)) * 2 + m) * kKeys + row) * D + col;
      const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
      x[0] += a.x, x[1] += a.y, x[2] += a.z, x[3] += a.w, x[4] += b.x, x[5] += b.y, x[6] += b.z, x[7] += b.w;
    }
    const float scale = m == 0 ? (BF16 ? 1.0f : 1.0f / 16384.0f) : p.scale * down;
    uint32_t v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = pack2<BF16>(x[2 * q] * scale, x[2 * q + 1] * scale);
    uint8_t* dst = static_cast<uint8_t*>(m == 0 ? p.dv : p.dk) + 2 * (((static_cast<size_t>(seq) * p.L + key) * p.kv_heads + kv_head) * p.d + col);
    *reinterpret_cast<uint4*>(dst) = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

}  // namespace

// ------------------------------------------------------------------ gradients of queries
template <int D, bool BF16, bool CAPPED, bool BIASED>
__global__ void __launch_bounds__(kThreads, 1) backward_queries_kernel(const __grid_constant__ BackwardParams p) {
  using LO = Layout<D>;
  constexpr int kAtoms = LO::kAtoms, kTile = LO::kTile, kHalfTile = LO::kHalfTile;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bar = reinterpret_cast<Bars*>(smem + LO::kOffBar);
  Segment<1>* segments = reinterpret_cast<Segment<1>*>(smem + LO::kOffSeg);
  static_assert(sizeof(Segment<1>) * kSegs <= 512, "segments");
  volatile uint32_t* abort_word = &bar->abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bar->keep_full, 1);
    mbar_init(&bar->keep_empty, 2);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 2);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&bar->s_full[g], 1);
      mbar_init(&bar->p_full[g], kComputeWarps / 2);
      mbar_init(&bar->dp_full[g], 1);
      mbar_init(&bar->ds_full[g], kComputeWarps / 2);
    }
    mbar_init(&bar->acc_done, 2);
    mbar_init(&bar->acc_free, kComputeWarps);
    mbar_init(&bar->sums_full, kComputeWarps);
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(&bar->seg_full[i], 1);
      mbar_init(&bar->seg_empty[i], kComputeWarps + 2);
    }
    bar->abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&bar->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = bar->tmem_base;
  grid_dependency_wait();
  grid_launch_dependents();

  if (warp == kProducerWarp) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const uint32_t half_bytes = static_cast<uint32_t>(p.half_rows) * 128 * kAtoms;
      DenseWalker<1> walker;
      Segment<1> s;
      int n = 0, keeps = 0;
      bool ok = true;
      for (int segs = 0; ok; ++segs) {
        bool more;
        do {
          more = walker.next(p, s);
        } while (more && s.seq < 0);
        const int slot = segs % kSegs;
        ok = mbar_wait(&bar->seg_empty[slot], ((segs / kSegs) & 1) ^ 1, abort_word, 0x120);
        if (!ok) break;
        s.valid = more;
        segments[slot] = s;
        mbar_arrive(&bar->seg_full[slot]);
        if (!more) break;
        if (s.lo0 >= s.hi0) continue;
        ok = mbar_wait(&bar->keep_empty, (keeps & 1) ^ 1, abort_word, 0x100);
        if (!ok) break;
        ++keeps;
        mbar_arrive_expect_tx(&bar->keep_full, 4 * half_bytes);
        load_halves<D>(smem + LO::kOffA, &p.map_q, &bar->keep_full, s.kv_head * p.group, p.head_step, s.first_token, p.half_tokens, s.seq);
        load_halves<D>(smem + LO::kOffB, &p.map_do, &bar->keep_full, s.kv_head * p.group, p.head_step, s.first_token, p.half_tokens, s.seq);
        for (int j = s.lo0; ok && j < s.hi0; ++j, ++n) {
          for (int g = 0; g < 2; ++g) {
            const int h = 2 * n + g, st = h & 3;
            ok = mbar_wait(&bar->empty[st], ((h >> 2) & 1) ^ 1, abort_word, 0x110);
            if (!ok) break;
            mbar_arrive_expect_tx(&bar->full[st], kTile);
            uint8_t* dst = smem + LO::kOffRing + st * kTile;
            for (int a = 0; a < kAtoms; ++a) {
              tma_load_4d(dst + a * (kHalf * 128), &p.map_k, &bar->full[st], a * 64, j * kKeys + g * kHalf, s.kv_head, s.seq);
              tma_load_4d(dst + kHalfTile + a * (kHalf * 128), &p.map_v, &bar->full[st], a * 64, j * kKeys + g * kHalf, s.kv_head, s.seq);
            }
          }
        }
      }
    }
  } else if (warp >= kMmaWarp) {
    // ------------------------------------------------------------ MMA: warp 0 S = Q K^T and P K, warp 1 dP = dO V^T and dS K
    issue_products<D, BF16>(smem, bar, tmem_base, segments, warp - kMmaWarp, lane, 0, [](const Segment<1>& s, int* lo, int* hi) { *lo = s.lo0, *hi = s.hi0; });
  } else {
    // ------------------------------------------------------------ arithmetic: thread a row and a quarter of the block's keys
    const int quad = warp & 3, part_of_row = warp >> 2, g = warp >> 3, row = quad * 32 + lane;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    const float c = p.c;
    float up, down;
    ds_scale<BF16>(p, &up, &down);
    const float p_down = BF16 ? 1.0f : 1.0f / 16384.0f, f = BF16 ? 1.0f : up * p_down;
    float* sums = reinterpret_cast<float*>(smem + LO::kOffRows);      // [2][4][128]: of dS, to set delta right
    const int r_half = row / kHalf, r_in = row % kHalf, r_token = r_half * p.half_tokens + r_in / p.half_heads,
              r_head = r_half * p.head_step + r_in % p.half_heads;
    const bool row_used = r_in < p.half_rows && r_head < p.group;
    int n = 0;
    uint32_t accs = 0;
    bool ok = true;
    for (int segs = 0;; ++segs) {
      const int slot = segs % kSegs;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar->seg_full[slot], (segs / kSegs) & 1, abort_word, 0x840));
      if (!ok) break;
      const Segment<1>& s = segments[slot];
      if (!s.valid) break;
      const int lo = s.lo0, hi = s.hi0, token = s.first_token + r_token, pos = token + s.keys - s.tokens;
      const bool valid = row_used && token < s.tokens;
      HalfRows& rows = p.rows[((static_cast<size_t>(s.seq) * p.kv_heads + s.kv_head) * p.tiles + s.first_token / p.tile_tokens) * 2 + r_half];
      const float off = rows.lse[r_in], delta = rows.delta[r_in], slope = BIASED ? rows.slope[r_in] : 0.f;
      int limit = valid ? visible_keys(pos, s.keys, p.causal, s.prefix) : 0, low = 0, doc = -1;
      bool mixed = false;
      if (p.documents != nullptr) {
        if (valid) {
          const size_t at = static_cast<size_t>(s.seq) * p.L + pos;
          const int2 run = p.runs[at];
          low = run.x;
          limit = min(limit, run.y);
          doc = p.documents[at];
        }
        mixed = p.mixed[s.seq] != 0;
      }
      uint64_t sum2 = 0;
      const int limit_of_all = __reduce_min_sync(0xffffffffu, limit), low_of_all = __reduce_max_sync(0xffffffffu, low);
      const bool behind = p.causal && s.prefix <= s.keys - s.tokens + s.first_token + 1;      // every key that a row sees is at or in front of it
      for (int j = lo; j < hi; ++j, ++n) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bar->s_full[g], n & 1, abort_word, 0x800));
        if (!ok) break;
        tc_fence_after_sync();
        const int k0 = j * kKeys + part_of_row * kCols;
        const bool cut = limit_of_all < k0 + kCols, cut_low = low_of_all > k0;
        float w[kCols] = {};
        [[maybe_unused]] float weight[CAPPED ? kCols : 1];      // without the cap's factor
        {
          uint32_t sv[32];
          tmem_ld_x32_wait(lane_base + kColS + part_of_row * kCols, sv);
          if constexpr (CAPPED) {
              capped(sv, p.cap_in, 1.0f);
              const uint64_t one2 = pack_f32x2(1.0f, 1.0f), out2 = pack_f32x2(p.cap_out, p.cap_out);
#pragma unroll
              for (int u = 0; u < 32; u += 2) {
                const uint64_t t = pack_f32x2(__uint_as_float(sv[u]), __uint_as_float(sv[u + 1]));
                unpack_f32x2(fma_f32x2(mul_f32x2(t, pack_f32x2(-1.0f, -1.0f)), t, one2), w[u], w[u + 1]);
                float y0, y1;
                unpack_f32x2(mul_f32x2(t, out2), y0, y1);
                sv[u] = __float_as_uint(y0), sv[u + 1] = __float_as_uint(y1);
              }
          }
          if constexpr (BIASED) {
            if (p.slopes != nullptr) biased(sv, CAPPED ? 1.0f : p.score_log2, -slope, static_cast<float>(pos - k0), behind);
          }
          if (mixed) {
            const int* ids = p.documents + static_cast<size_t>(s.seq) * p.L;
#pragma unroll
            for (int u = 0; u < 32; ++u) {
              if (ids[min(k0 + u, p.L - 1)] != doc) sv[u] = __float_as_uint(-INFINITY);
              if (u % 8 == 7) asm volatile("" ::: "memory");       // (eight ids at a time: registers)
            }
          }
          if (cut_low) {
#pragma unroll
            for (int u = 0; u < 32; ++u)
              if (u < low - k0) sv[u] = __float_as_uint(-INFINITY);
          }
          if (cut) {
            const int lim = limit - k0;
#pragma unroll
            for (int u = 0; u < 32; ++u)
              if (u >= lim) sv[u] = __float_as_uint(-INFINITY);
          }
          const uint64_t c2 = pack_f32x2(c, c), off2 = pack_f32x2(off, off);
          uint32_t pk[16];
#pragma unroll
          for (int u = 0; u < 32; u += 2) {
            uint64_t x = softmax_weights(sv[u], sv[u + 1], c2, off2, false);
            if constexpr (CAPPED) {
              unpack_f32x2(x, weight[u], weight[u + 1]);
              x = mul_f32x2(x, pack_f32x2(w[u], w[u + 1]));
            }
            float p0, p1;
            unpack_f32x2(x, p0, p1);
            pk[u / 2] = pack2<BF16>(p0, p1);
            if constexpr (!BF16) x = mul_f32x2(x, pack_f32x2(f, f));
            unpack_f32x2(x, w[u], w[u + 1]);
          }
          tmem_st_x16(lane_base + kColS + part_of_row * kCols, pk);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive_warp(&bar->p_full[g], lane);

        ok = __all_sync(0xffffffffu, mbar_wait(&bar->dp_full[g], n & 1, abort_word, 0x810));
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t dp_col = lane_base + kColDp + part_of_row * kCols;
        const uint64_t delta2 = pack_f32x2(delta, delta);
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += 16) {
          uint32_t dp[16], pk[8];
          tmem_ld_x16_wait(dp_col + c0, dp);
#pragma unroll
          for (int u = 0; u < 16; u += 2) {
            const uint64_t d = add_f32x2(pack_f32x2(__uint_as_float(dp[u]), __uint_as_float(dp[u + 1])), delta2),
                           x = mul_f32x2(pack_f32x2(w[c0 + u], w[c0 + u + 1]), d);
            if constexpr (CAPPED) sum2 = fma_f32x2(pack_f32x2(weight[c0 + u], weight[c0 + u + 1]), d, sum2);
            else sum2 = add_f32x2(sum2, x);
            float x0, x1;
            unpack_f32x2(x, x0, x1);
            pk[u / 2] = pack2<BF16>(x0, x1);
          }
          tmem_st_x8(dp_col + c0 / 2, pk);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive_warp(&bar->ds_full[g], lane);
      }
      if (!ok) break;

      const bool has = lo < hi;
      if (has) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bar->acc_done, accs & 1, abort_word, 0x830));
        ++accs;
        if (!ok) break;
        tc_fence_after_sync();
      }
      // What delta is off by: the sum of the row's P (dP - delta), which is 0 for the right one.  delta comes from a result that is rounded, and
      // was summed from rounded weights: a step of the type relative to a difference that can be small beside it where few keys have the weight.
      // dS misses -P times that (and the cap's factor), so dQ misses it times P K; the keys' kernel, behind this one, gets delta set right.
      float s0, s1;
      unpack_f32x2(sum2, s0, s1);
      float* mine = sums + (segs & 1) * 512 + row;
      mine[part_of_row * 128] = s0 + s1;
      mbar_arrive_warp(&bar->sums_full, lane);
      ok = __all_sync(0xffffffffu, mbar_wait(&bar->sums_full, segs & 1, abort_word, 0x850));
      if (!ok) break;
      const float off_by = (mine[0] + mine[128] + mine[256] + mine[384]) * (CAPPED ? p_down : down);
      if (part_of_row == 0 && valid) rows.delta[r_in] = delta - off_by;
      // (a row that sees one key: nothing, and not what rounding leaves of it; the keys' dS is 0 by itself, delta being dP)
      const bool lone = !mixed && limit - low == 1;
      const float scale = lone ? 0.f : p.scale * down, scale_pk = lone ? 0.f : -p.scale * off_by * p_down;
      uint8_t* dst = static_cast<uint8_t*>(p.dq) + 2 * ((static_cast<size_t>(s.seq) * p.M + token) * p.heads + s.kv_head * p.group + r_head) * p.d;
#pragma unroll
      for (int cc = 0; cc < D / 4; cc += 16) {
        const int col = part_of_row * (D / 4) + cc;
        float x[16];
        if (has) {
          uint32_t ds[16], pk[16];
          tmem_ld_x16_wait(lane_base + kColAcc + D + col, ds);
          tmem_ld_x16_wait(lane_base + kColAcc + col, pk);
#pragma unroll
          for (int u = 0; u < 16; ++u) x[u] = fmaf(__uint_as_float(pk[u]), scale_pk, __uint_as_float(ds[u]) * scale);
        } else {
#pragma unroll
          for (int u = 0; u < 16; ++u) x[u] = 0.f;
        }
        if (cc + 16 == D / 4) {
          tc_fence_before_sync();
          if (has) mbar_arrive_warp(&bar->acc_free, lane);
        }
        if (!valid) continue;
#pragma unroll
        for (int u = 0; u < 16; u += 8) {
          uint32_t v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = pack2<BF16>(x[u + 2 * q], x[u + 2 * q + 1]);
          if (col + u < p.d) *reinterpret_cast<uint4*>(dst + 2 * (col + u)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
      mbar_arrive_warp(&bar->seg_empty[slot], lane);
    }
  }

  if (bar->abort_word != 0u) {
    for (int t = 0; t < 64; ++t) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tmem_dealloc(tmem_base, kTmemCols);
    if (lane == 0 && bar->abort_word != 0 && p.status != nullptr) atomicCAS(p.status, 0, static_cast<int>(bar->abort_word));
  }
}

namespace {

cudaLaunchConfig_t config(long long grid, int threads, int smem, cudaStream_t stream, cudaLaunchAttribute* attr, int slices = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), static_cast<unsigned>(slices), 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

template <int D, bool BF16, bool CAPPED, bool BIASED>
cudaError_t launch_products(const BackwardParams& p, int sms, cudaStream_t stream) {
  auto keys = backward_keys_kernel<D, BF16, CAPPED, BIASED>;
  auto queries = backward_queries_kernel<D, BF16, CAPPED, BIASED>;
  static std::atomic<unsigned long long> configured{0};
  int dev = 0;
  cudaError_t e = current_device_checked(&dev);
  if (e != cudaSuccess) return e;
  if (!device_configured(configured, dev)) {
    e = cudaFuncSetAttribute(keys, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kBytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(queries, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kBytes);
    if (e != cudaSuccess) return e;
    mark_device_configured(configured, dev);
  }
  cudaLaunchAttribute attr[1];
  e = launch_kernel(config(p.items < sms ? p.items : sms, kThreads, Layout<D>::kBytes, stream, attr), queries, p);      // (sets delta right)
  if (e == cudaSuccess) e = launch_kernel(config(sms, kThreads, Layout<D>::kBytes, stream, attr), keys, p);
  if (e == cudaSuccess) e = launch_kernel(config(sms, kSumThreads, 0, stream, attr, kSumSlices), sum_key_parts_kernel<D, BF16>, p);
  return e;
}

}  // namespace

template <int D, bool BF16>
cudaError_t launch_backward(const BackwardParams& p, int sms, cudaStream_t stream) {
  if (!BF16) {
    const cudaError_t e = cudaMemsetAsync(p.norms, 0, 2 * sizeof(uint32_t), stream);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t rows = config(2 * p.items < 16 * sms ? 2 * p.items : 16 * sms, kRowThreads, 0, stream, attr);
  const cudaError_t e = D == 64 ? launch_kernel(rows, backward_rows_kernel<BF16, 8>, p) : launch_kernel(rows, backward_rows_kernel<BF16, 16>, p);
  if (e != cudaSuccess) return e;
  if (p.cap_out != 0.f) return launch_products<D, BF16, true, true>(p, sms, stream);      // (with slopes or without)
  return p.slopes != nullptr ? launch_products<D, BF16, false, true>(p, sms, stream) : launch_products<D, BF16, false, false>(p, sms, stream);
}

template cudaError_t launch_backward<(DITTO_MASKED_BACKWARD_PART & 1) ? 128 : 64, (DITTO_MASKED_BACKWARD_PART & 2) != 0>(const BackwardParams&, int,
                                                                                                                       cudaStream_t);

}  // namespace masked
}  // namespace ditto_b200
