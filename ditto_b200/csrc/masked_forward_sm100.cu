// Forward kernel of the masked attention operators: dense items, and chunks or single tokens over a paged cache.
//
// For a row i with scores s_ij (capped, biased) over the keys j that it sees: O_i = sum_j 2^(c s_ij - m_i) V_j / l_i in one pass with
// the running reference m_i and sum l_i, lse_i = ln(2) (m_i + log2 l_i).
//
// A CTA walks items of one or two 128-row tiles.  A step is a tile and a block of 128 keys: S = Q K^T into one of two 128-column buffers
// of tensor memory, P over the scores by the four warps that belong to the buffer (a thread a row), O += P V into the buffer's own
// accumulator.  Two tiles: a buffer each, and each K/V block is loaded once for both.  One tile: its blocks go to the buffers in turn and
// the two accumulators are joined at the end.  A step goes in halves of 64 keys, so that a half's scores are computed under the other half's
// exponentials and a thread holds 64 scores, which leave it room to compute with.  Each buffer has an MMA warp of its own: issuing waits for
// room in the tensor pipe's queue, and with one warp for both its bookkeeping left the pipe idle for 900 of 2450 clocks a step.
//
// What bounds it: the exponentials and what stands around them.  With heads of 64 the tensor pipe is busy for 27 % of the time, the
// special-function unit for about half of it and an instruction issued in 40 % of the clocks: two warps a scheduler do not cover each
// other's latencies, and there are registers for no more.  16 heads, 8192 x 8192, bf16: d = 128 full 529 us (1040 TFLOP/s), causal 252
// us (1090); d = 64 full 489 us (563), causal 230 us (597).  Causal with a cap 373 us, with a bias by distance 300 us.
//
// Over a paged cache the blocks of all items are dealt out to the CTAs in equal shares, whatever the sequences' lengths: an item that a
// share cuts is finished by a second kernel from fp32 parts.  8192 tokens over 16384 keys, 16 heads over two of 128, biased: 809 us for this
// kernel, 19 us for the second; with single tokens it is bound by its reads (SPLIT, below).
#include <atomic>

#include "host_util.cuh"
#include "masked_sm100.cuh"
#include "mlp_common.cuh"
#include "sm100_ptx.cuh"
#include "softmax_step.cuh"

#ifndef DITTO_MASKED_PART
#define DITTO_MASKED_PART 0
#endif

namespace ditto_b200 {
namespace masked {
namespace {

constexpr int kSoftmaxWarps = 8, kThreads = 32 * (kSoftmaxWarps + 3);
constexpr int kProducerWarp = kSoftmaxWarps, kMmaWarp = kSoftmaxWarps + 1;      // (and the one behind it: a warp a buffer)
constexpr uint32_t kTmemCols = 512, kColO = 256;
constexpr float kRescaleThreshold = 8.0f;     // log2 units by which a row's maximum may run ahead of its reference
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kSegs = 4;                      // items that the producer is ahead of the others

// SPLIT: items of a single token, whose heads (32 at most) fill a part of a tile only.  Four copies of the rows, at rows 0, 32, 64 and 96: a warp has
// a quarter of a block's keys of each row instead of a thread a whole row, and no weight on the others; the copies' results are summed at an item's
// end.  A block takes a quarter of the time, below that of its loads.  64 ragged sequences of up to 16384 keys, 32 heads over 8 of 128: 414 -> 363 us
// (6.0 TB/s), of 64, 128 sequences: 730 -> 425 us (5.8 TB/s).
template <int D, int NT, bool SPLIT>
struct Layout {
  static constexpr int kAtoms = D / 64;
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kStages = D == 128 ? (NT == 2 || SPLIT ? 4 : 5) : 8;     // K and V blocks in turn
  static constexpr int kOffKV = NT * kTile;
  static constexpr int kOffBias = kOffKV + kStages * kTile;            // what the product of the bias reads
  static constexpr int kOffSum = kOffBias + kRows * 128;               // [2][buffer][128] references and sums
  static constexpr int kOffJoin = kOffSum + 4096;                      // (SPLIT) [2][warp][32 rows][16] of the accumulators
  static constexpr int kOffBar = kOffJoin + (SPLIT ? 2 * kSoftmaxWarps * 2048 : 0);
  static constexpr int kOffSeg = kOffBar + 1024;
  static constexpr int kBytes = kOffSeg + 512 + 1024;
};

struct Bars {
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[8], kv_empty[8];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2], o_done[2], o_free[2];      // [buffer][half]
  uint64_t seg_full[kSegs], seg_empty[kSegs];
  uint64_t sums_full, join_full;
  uint32_t tmem_base, abort_word;
  PagedStart start;
  int scan[kThreads / 32 + 1];
};
static_assert(sizeof(Bars) <= 1024, "barrier block too large");

// The bias by distance as a 16-wide step more of the scores' product, for rows that see no key behind them: -slope (pos - k0 - i) is
// slope i, which the step adds, plus a number per row and block, slope (k0 - pos), which goes into the row's maximum and the exponents' offset.
// The step's rows hold the slope (over the scale) as a sum of three bf16, 24 bits; its columns the key's place i in the block three times, which
// bf16 holds exactly.  One buffer of 128 rows of 128 bytes, swizzled like the tiles: the slopes of tile 0 in bytes 0 to 31 of a row, those of tile 1 in
// 32 to 63, the places in 64 to 95.  Element by element the bias took 540 us of the same work that takes 300 now.
__device__ __forceinline__ uint8_t* bias_at(uint8_t* buffer, int row, int sixteenths) { return buffer + row * 128 + ((sixteenths ^ (row & 7)) << 4); }
__device__ __forceinline__ uint2 bias_terms(float x) {
  const __nv_bfloat16 a = __float2bfloat16(x);
  x -= __bfloat162float(a);
  const __nv_bfloat16 b = __float2bfloat16(x);
  x -= __bfloat162float(b);
  const __nv_bfloat16 c = __float2bfloat16(x);
  return make_uint2(__bfloat16_as_ushort(a) | static_cast<uint32_t>(__bfloat16_as_ushort(b)) << 16, __bfloat16_as_ushort(c));
}
// Whether every key that a row of tile t sees is at or in front of it.
template <int NT>
__device__ __forceinline__ bool keys_in_front(const Params& p, const Segment<NT>& s, int t) {
  return p.causal && s.prefix <= s.keys - s.tokens + s.first_token + t * p.tile_tokens + 1;
}

// Shares of a paged call: the blocks of all items of a lane of heads, in order, in gridDim.x / lanes equal shares.
template <int NT>
__device__ __forceinline__ void find_start(const Params& p, Bars* bar) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kWarps = kThreads / 32;
  const int heads = p.kv_heads / p.lanes;
  int mine = 0, first_cost = 0;
  for (int b = tid; b < p.batch; b += kThreads) {
    Sequence q;
    q.load(p, b);
    const int cost = heads * q.template units_of_head<NT>(p);
    if (b == tid) first_cost = cost;
    mine += cost;
  }
  int sum = mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) bar->scan[warp] = sum;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < kWarps; ++w) total += bar->scan[w];
  const int shares = gridDim.x / p.lanes, per = max(1, (total + shares - 1) / shares);
  const int u0 = min(static_cast<long long>(per) * (blockIdx.x / p.lanes), static_cast<long long>(total)), left = min(per, total - u0);
  if (tid == 0) bar->start = {0, 0, 0, 0, 0, per};
  int before = 0;                                  // blocks of the sequences of earlier rounds
  for (int base = 0; base < p.batch; base += kThreads) {
    const int b = base + tid;
    Sequence q;
    int cost = first_cost;
    if (base > 0) {
      cost = 0;
      if (b < p.batch) {
        q.load(p, b);
        cost = heads * q.template units_of_head<NT>(p);
      }
    }
    int incl = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();                               // the scratch of the round before is free
    if (lane == 31) bar->scan[warp] = incl;
    __syncthreads();
    int offset = before, all = before;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) offset += bar->scan[w];
      all += bar->scan[w];
    }
    const int at = u0 - (offset + incl - cost);    // inside this thread's sequence?
    if (left > 0 && at >= 0 && at < cost) {
      q.load(p, b);
      const int of_head = cost / heads;
      PagedStart s = {b, at / of_head, 0, at % of_head, left, per};
      for (int n; (n = q.template units<NT>(p, s.first_token)) <= s.block; s.first_token += NT * p.tile_tokens) s.block -= n;
      bar->start = s;
    }
    before = all;
  }
  __syncthreads();
}

}  // namespace

template <int D, bool BF16, int NT, bool PAGED, bool CAPPED, bool BIASED, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) masked_forward_kernel(const __grid_constant__ Params p) {
  using LO = Layout<D, NT, SPLIT>;
  static_assert(!SPLIT || (NT == 1 && PAGED), "four copies of an item's rows: single tokens");
  constexpr int kStages = LO::kStages, kAtoms = LO::kAtoms, kTile = LO::kTile;
  constexpr bool kBiasProduct = BIASED && !CAPPED;
  // a block's scores and weights come in halves, the next one's scores under the other's weights; single tokens' wait for memory, not for these
  constexpr int kPieces = SPLIT ? 1 : 2, kPiece = kKeys / kPieces;
  // Biased scores grow along a row, by 184 slope a block in units of the exponent: taken from the last block to the first, hardly a row has
  // to move its reference, and its accumulator with it, more than once.  (Causal, 16 heads of 128 over 8192 tokens: 292 us instead of 356.)
  constexpr bool kBack = kBiasProduct;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bar = reinterpret_cast<Bars*>(smem + LO::kOffBar);
  volatile uint32_t* abort_word = &bar->abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->q_full[i], 1);
      mbar_init(&bar->q_empty[i], NT == 2 ? 1 : 2);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bar->s_full[i][h], 1);
        mbar_init(&bar->p_full[i][h], kSoftmaxWarps / 2);
      }
      mbar_init(&bar->pv_done[i], 1);
      mbar_init(&bar->o_done[i], 1);
      mbar_init(&bar->o_free[i], NT == 2 ? kSoftmaxWarps / 2 : kSoftmaxWarps);
    }
    mbar_init(&bar->sums_full, kSoftmaxWarps);
    mbar_init(&bar->join_full, kSoftmaxWarps);
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(&bar->seg_full[i], 1);
      mbar_init(&bar->seg_empty[i], kSoftmaxWarps + 2);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar->kv_full[i], 1);
      mbar_init(&bar->kv_empty[i], NT);
    }
    bar->abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&bar->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  if constexpr (kBiasProduct) {
    uint8_t* bias = smem + LO::kOffBias;
    for (int i = threadIdx.x; i < kRows * 8; i += kThreads) {
      const int row = i >> 3, piece = i & 7;
      const uint32_t place = __bfloat16_as_ushort(__int2bfloat16_rn(row));
      *reinterpret_cast<uint4*>(bias_at(bias, row, piece)) = piece == 4 ? make_uint4(place | place << 16, place, 0, 0) : make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
  }
  if (warp == kProducerWarp && lane == 0) {
    tma_prefetch_desc(&p.map_q);
    tma_prefetch_desc(&p.map_k);
    tma_prefetch_desc(&p.map_v);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = bar->tmem_base;
  grid_dependency_wait();
  grid_launch_dependents();

  if constexpr (PAGED) {
    if (!p.whole) {
      find_start<NT>(p, bar);
    } else {
      if (threadIdx.x == 0) bar->start = {0, 0, 0, 0, 0, 0};
      __syncthreads();
    }
  }
  // The producer finds the items and hands them to the others through shared memory (the registers of the softmax warps are for scores).
  Segment<NT>* segments = reinterpret_cast<Segment<NT>*>(smem + LO::kOffSeg);
  static_assert(sizeof(Segment<NT>) * kSegs <= 512, "segments");

  if (warp == kProducerWarp) {
    // ------------------------------------------------------------ TMA producer (converged; lane 0, or a lane a page, issues)
    auto w = [&]() {
      if constexpr (PAGED) {
        return PagedWalker<NT>(bar->start);
      } else {
        return DenseWalker<NT>();
      }
    }();
    Segment<NT> s;
    int g = 0, segs = 0;
    uint32_t loads_q = 0;                          // parities, a bit a tile
    bool ok = true;
    const uint32_t q_bytes = static_cast<uint32_t>(p.group * p.tile_tokens) * 128 * kAtoms * (SPLIT ? 4 : 1);
    bool more = true;
    while (ok && more) {
      do {
        more = w.next(p, s);
      } while (more && s.seq < 0);
      const int slot = segs % kSegs;
      ok = __all_sync(0xffffffffu, mbar_wait(&bar->seg_empty[slot], ((segs / kSegs) & 1) ^ 1, abort_word, 0x120));
      if (!ok) break;
      if (lane == 0) {
        s.valid = more;
        s.block0 = g;
        segments[slot] = s;
        mbar_arrive(&bar->seg_full[slot]);
      }
      __syncwarp();
      ++segs;
      if (!more) break;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (!ok || s.lo(t) >= s.hi(t)) continue;
        ok = __all_sync(0xffffffffu, mbar_wait(&bar->q_empty[t], ((loads_q >> t) & 1) ^ 1, abort_word, 0x100 + t));
        if (!ok) break;
        loads_q ^= 1u << t;
        if constexpr (kBiasProduct) {
          const bool brought = p.bias_product && keys_in_front(p, s, t);
          for (int row = lane; row < kRows; row += 32) {
            const float slope = brought ? p.slopes[s.kv_head * p.group + (SPLIT ? row % 32 : row) % p.group] * p.bias_unit : 0.f;
            *reinterpret_cast<uint2*>(bias_at(smem + LO::kOffBias, row, 2 * t)) = bias_terms(slope);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&bar->q_full[t], q_bytes);
          for (int copy = 0; copy < (SPLIT ? 4 : 1); ++copy)
           for (int a = 0; a < kAtoms; ++a)
            tma_load_4d(smem + t * kTile + a * (kRows * 128) + copy * (32 * 128), &p.map_q, &bar->q_full[t], a * 64, s.kv_head * p.group,
                        s.row0 + s.first_token + t * p.tile_tokens, PAGED ? 0 : s.seq);
        }
        __syncwarp();
      }
      // lane l's entry of the table for step i, read a step ahead: page l of the block
      const int page_rows = PAGED ? min(p.page, kKeys) : kKeys;
      auto pages_of = [&](int j) { return min(kKeys / page_rows, (s.keys - j * kKeys + page_rows - 1) / page_rows); };
      auto entry = [&](int i) {
        const int j = s.template block<kBack>(i);
        return lane < pages_of(j) ? p.table[s.seq * p.table_stride + (j * kKeys + lane * page_rows) / p.page] : -1;
      };
      [[maybe_unused]] int ahead = PAGED && s.begin() < s.end() ? entry(s.begin()) : -1;
      for (int i = s.begin(); ok && i < s.end(); ++i) {
        const int j = s.template block<kBack>(i);
        // rows of this block that pages bring: lane i loads page i of the block
        const int rows = page_rows;
        int page = -1, lanes = 1, row_in_page = 0;
        if constexpr (PAGED) {
          lanes = pages_of(j);
          row_in_page = (j * kKeys) % p.page;          // (0 unless a page is longer than a block)
          page = ahead;
          if (i + 1 < s.end()) ahead = entry(i + 1);
          if (lane < lanes) {
            if (page < 0 || page >= p.pages) {
              page = -1;                               // (out of the map's range: zeros)
              if (p.status != nullptr) atomicCAS(p.status, 0, kBadPage);
            }
          }
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int n = 2 * g + kv, st = n % kStages;
          ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar->kv_empty[st], ((n / kStages) & 1) ^ 1, abort_word, 0x110 + kv));
          if (!ok) break;
          const CUtensorMap* map = kv == 0 ? &p.map_k : &p.map_v;
          uint8_t* dst = smem + LO::kOffKV + st * kTile;
          if (lane == 0) mbar_arrive_expect_tx(&bar->kv_full[st], static_cast<uint32_t>(lanes * rows) * 128 * kAtoms);
          __syncwarp();
          if (lane < lanes) {
            for (int a = 0; a < kAtoms; ++a) {
              if constexpr (PAGED)
                tma_load_4d(dst + a * (kKeys * 128) + lane * rows * 128, map, &bar->kv_full[st], a * 64, row_in_page, s.kv_head, page);
              else
                tma_load_4d(dst + a * (kKeys * 128), map, &bar->kv_full[st], a * 64, j * kKeys, s.kv_head, s.seq);
            }
          }
          __syncwarp();
        }
        ++g;
      }
    }
  } else if (warp >= kMmaWarp) {
    // ------------------------------------------------------------ MMA issuer of a buffer (converged warp, elected lane issues)
    const int buf = warp - kMmaWarp, t = NT == 2 ? buf : 0;
    const uint32_t issuer = elect_one();
    const uint32_t idesc_s = umma_idesc_f16(BF16, kRows, kPiece, false, false);
    const uint32_t idesc_o = umma_idesc_f16(BF16, kRows, D, false, true);
    const uint64_t dq = umma_desc_sw128(smem_u32(smem + t * kTile), 16, 1024);
    const uint64_t dk0 = umma_desc_sw128(smem_u32(smem + LO::kOffKV), 16, 1024);
    const uint64_t dv0 = umma_desc_sw128(smem_u32(smem + LO::kOffKV), kKeys * 128, 1024);
    [[maybe_unused]] const uint32_t idesc_bias = umma_idesc_f16(true, kRows, kPiece, false, false);
    [[maybe_unused]] const uint64_t dbias = umma_desc_sw128(smem_u32(smem + LO::kOffBias), 16, 1024);
    const uint32_t d_o = tmem_base + kColO + buf * D, d_s = tmem_base + buf * kKeys;
    auto wait = [&](uint64_t* b, uint32_t parity, uint32_t code) {
      const bool r = __all_sync(0xffffffffu, mbar_wait(b, parity, abort_word, code));
      tc_fence_after_sync();
      return r;
    };
    // (of two barriers at once: a vote and a fence less)
    auto wait_both = [&](uint64_t* b, uint32_t parity, uint64_t* b2, uint32_t parity2, uint32_t code) {
      const bool r = __all_sync(0xffffffffu, mbar_wait(b, parity, abort_word, code) && mbar_wait(b2, parity2, abort_word, code));
      tc_fence_after_sync();
      return r;
    };
    auto wait_kv = [&](int n) { return wait(&bar->kv_full[n % kStages], (n / kStages) & 1, 0x310); };      // n: 2 block, or 2 block + 1
    auto issue_s = [&](int block, int h) {
      const int st = (2 * block) % kStages;
      const uint64_t db = dk0 + ((st * kTile + h * (kPiece * 128)) >> 4);
      const uint32_t d = d_s + h * kPiece;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint32_t off = ((i / 4) * (kRows * 128) + (i % 4) * 32) >> 4;
        umma_ss_elected(d, dq + off, db + off, idesc_s, i > 0 ? 1u : 0u, issuer);
      }
      if constexpr (kBiasProduct) umma_ss_elected(d, dbias + 2 * t, dbias + 4 + ((h * (kPiece * 128)) >> 4), idesc_bias, 1u, issuer);
      umma_commit_elected(&bar->s_full[buf][h], issuer);
      if (h == kPieces - 1) umma_commit_elected(&bar->kv_empty[st], issuer);
    };
    constexpr int kStep = NT == 2 ? 1 : 2;
    uint32_t loads_q = 0, uses_o = 0, n = 0;           // tiles and accumulators so far, steps so far
    bool ok = true;
    for (int segs = 0; ok; ++segs) {
      const int slot = segs % kSegs;
      ok = wait(&bar->seg_full[slot], (segs / kSegs) & 1, 0x350);
      if (!ok || !segments[slot].valid) break;
      const int begin = segments[slot].begin(), end = segments[slot].end(), block0 = segments[slot].block0 - begin;
      const int first = segments[slot].template first_step<kBack>(t) + (NT == 1 ? buf : 0), last = segments[slot].template last_step<kBack>(t);
      if (begin >= end) {
        mbar_arrive_warp(&bar->seg_empty[slot], lane);
        continue;
      }
      // (two tiles) blocks that this tile does not see, for documents or causal masks, are released once they are there
      auto pass = [&](int j) {
        for (int kv = 0; kv < 2; ++kv) {
          if (!wait_kv(2 * (block0 + j) + kv)) return false;
          mbar_arrive_warp(&bar->kv_empty[(2 * (block0 + j) + kv) % kStages], lane);
        }
        return true;
      };
      if constexpr (NT == 2) {
        for (int j = begin; ok && j < min(first, end); ++j) ok = pass(j);
      }
      if (ok && (NT == 1 || first < last)) {
        ok = wait(&bar->q_full[t], loads_q & 1, 0x300 + t);
        ++loads_q;
      }
      if (!ok) break;
      if (first < last) {
        ok = wait_kv(2 * (block0 + first));
        if (!ok) break;
        for (int h = 0; h < kPieces; ++h) issue_s(block0 + first, h);
      }
      mbar_arrive_warp(&bar->seg_empty[slot], lane);
      if (first + kStep >= last) {                     // Q has been read with the item's last scores
        if (first < last) umma_commit_elected(&bar->q_empty[t], issuer);
        else if (NT == 1 && lane == 0) mbar_arrive(&bar->q_empty[t]);
      }
      for (int j = first; j < last; j += kStep, ++n) {
        const int next = j + kStep, nv = 2 * (block0 + j) + 1, sv = nv % kStages;
        // What is most likely there is waited for first.  With one tile the next keys are waited for behind P V: they may still be on
        // their way where memory is the bound, and the values' place in the ring is wanted back.
        if (NT == 2 && next < last) {
          const int nk = 2 * (block0 + next);
          if (!(ok = wait_both(&bar->kv_full[sv], (nv / kStages) & 1, &bar->kv_full[nk % kStages], (nk / kStages) & 1, 0x310))) break;
        } else {
          if (!(ok = wait_kv(nv))) break;
        }
        if (j == first) {                              // a new accumulator: what it held has been read
          if (!(ok = wait(&bar->o_free[buf], (uses_o & 1) ^ 1, 0x320))) break;      // (at once the first time)
          ++uses_o;
        }
        const uint64_t db = dv0 + ((sv * kTile) >> 4);
        auto issue_pv = [&](int h) {
#pragma unroll
          for (int i = 0; i < kPiece / 16; ++i)
            umma_ts_elected(d_o, d_s + h * kPiece + i * 8, db + (((h * (kPiece / 16) + i) * 2048) >> 4), idesc_o, i > 0 || h > 0 || j > first ? 1u : 0u, issuer);
          umma_commit_elected(&bar->pv_done[buf], issuer);
        };
        if (!(ok = wait(&bar->p_full[buf][0], n & 1, 0x340))) break;
        issue_pv(0);
        if (NT == 2 && next < last) issue_s(block0 + next, 0);
        if constexpr (kPieces == 2) {
          if (!(ok = wait(&bar->p_full[buf][1], n & 1, 0x341))) break;
          issue_pv(1);
        }
        umma_commit_elected(&bar->kv_empty[sv], issuer);
        if (next < last) {
          if (NT == 1) {
            if (!(ok = wait_kv(2 * (block0 + next)))) break;
            issue_s(block0 + next, 0);
          }
          if (kPieces == 2) issue_s(block0 + next, 1);
          if (next + kStep >= last) umma_commit_elected(&bar->q_empty[t], issuer);
        } else {
          umma_commit_elected(&bar->o_done[buf], issuer);
        }
      }
      if constexpr (NT == 2) {
        for (int j = max(begin, max(last, min(first, end))); ok && j < end; ++j) ok = pass(j);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax: warps 0-3 buffer 0, 4-7 buffer 1; a thread a row
    const int quad = warp & 3, buf = warp >> 2, row = quad * 32 + lane;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t s_col = lane_base + buf * kKeys, o_col = lane_base + kColO;
    float2* sums = reinterpret_cast<float2*>(smem + LO::kOffSum) + row;
    const int in_copy = SPLIT ? lane : row, r_token = in_copy / p.group, r_head = in_copy - r_token * p.group;
    // this thread's keys of a block
    constexpr int kMine = SPLIT ? 32 : kPiece;
    const bool row_used = r_token < p.tile_tokens;
    const float c = p.c;
    const int t = NT == 2 ? buf : 0;
    int n = 0, segs = 0;
    [[maybe_unused]] int joins = 0;
    uint32_t done = 0;
    bool ok = true;
    if constexpr (PAGED) {
      if (threadIdx.x == 0) p.parts[blockIdx.x].last_cta = -1;
    }
    for (;; ++segs) {
      const int slot = segs % kSegs;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar->seg_full[slot], (segs / kSegs) & 1, abort_word, 0x840));
      if (!ok) break;
      const Segment<NT>& s = segments[slot];
      if (!s.valid) break;
      const int token = s.first_token + t * p.tile_tokens + r_token, pos = token + s.keys - s.tokens;
      const bool valid = row_used && token < s.tokens;
      const int head = s.kv_head * p.group + r_head;
      // the row sees keys from low up to limit; documents in another order than rising: those of them that have its id
      int limit = valid ? visible_keys(pos, s.keys, p.causal, s.prefix) : 0, low = 0, doc = -1;
      bool mixed = false;
      if constexpr (!PAGED) {
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
      }
      const float slope = BIASED && p.slopes != nullptr && valid ? p.slopes[head] * (CAPPED ? 1.4426950408889634f : p.bias_unit) : 0.f;
      // the first block that a row of this warp does not see whole, and the last one in which one does not see the first key (documents)
      const int cut = __reduce_min_sync(0xffffffffu, limit), cut_low = __reduce_max_sync(0xffffffffu, low);
      const bool in_front = keys_in_front(p, s, t), brought = kBiasProduct && p.bias_product && in_front;
      RowReference ref(c);
      if (limit == 0) ref.m = 0.f, ref.large = false;      // sees nothing: asks for no rescale
      float l = 0.f;
      const int first = s.template first_step<kBack>(t) + (NT == 1 ? buf : 0), end = s.template last_step<kBack>(t);
      for (int step = first; ok && step < end; step += NT == 1 ? 2 : 1, ++n) {
#pragma unroll 1                                       // (unrolled 6 to 18 % slower: twice the code)
       for (int h = 0; h < kPieces; ++h) {
        const int part0 = SPLIT ? quad * 32 : h * kPiece;       // this thread's keys of the block begin there
        ok = __all_sync(0xffffffffu, mbar_wait(&bar->s_full[buf][h], n & 1, abort_word, 0x800));
        if (!ok) break;
        tc_fence_after_sync();
        const int j = s.template block<kBack>(step), k0 = j * kKeys + part0;
        uint32_t sv[kMine];
        if constexpr (SPLIT) tmem_ld_x32_wait(s_col + part0, sv);
        else tmem_ld_x64_wait(s_col + part0, sv);
        float base = 0.f;                              // what the row's scores in sv lack
        if constexpr (CAPPED) {
          capped(sv, p.cap_in, p.cap_out);
          if (p.slopes != nullptr) biased(sv, 1.0f, slope, static_cast<float>(pos - k0), in_front);
        }
        if constexpr (kBiasProduct) {
          if (brought) base = slope * static_cast<float>(j * kKeys - pos);
          else biased(sv, p.bias_factor, slope, static_cast<float>(pos - k0), in_front);
        }
        if constexpr (!PAGED) {
          if (mixed) {
            const int* ids = p.documents + static_cast<size_t>(s.seq) * p.L;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
              if (ids[min(k0 + i, p.L - 1)] != doc) sv[i] = __float_as_uint(-INFINITY);
              if (i % 8 == 7) asm volatile("" ::: "memory");       // (eight ids at a time: registers)
            }
          }
        }
        if (k0 + kMine > cut) {
          const int lim = limit - k0;
#pragma unroll
          for (int i = 0; i < kMine; ++i)
            if (i >= lim) sv[i] = __float_as_uint(-INFINITY);
        }
        if (!PAGED && cut_low > k0) {
#pragma unroll
          for (int i = 0; i < kMine; ++i)
            if (i < low - k0) sv[i] = __float_as_uint(-INFINITY);
        }
        // Two tiles, items of many blocks: the weights against the reference so far, and the maximum beside them; it is seldom that it has to move,
        // and they are taken again.  (16 heads of 64, 8192 x 8192: 486 us instead of 507.)
        constexpr bool kAhead = NT == 2;
        uint32_t pk[kMine / 2];
        uint64_t sum2[2];
        auto weigh = [&]() {
          // (a reference far from 0 for the distance alone is near the row's scores in sv: the difference first)
          const float mc = kBiasProduct && !ref.large ? (ref.m - base) * c : ref.offset(c);
          const uint64_t c2 = pack_f32x2(c, c), nmc2 = pack_f32x2(-mc, -mc);
          sum2[0] = sum2[1] = 0;
#pragma unroll
          for (int i = 0; i < kMine / 2; ++i) {
            const uint64_t weights = softmax_weights(sv[2 * i], sv[2 * i + 1], c2, nmc2, weights_on_fma(i));
            sum2[i & 1] = add_f32x2(sum2[i & 1], weights);
            float p0, p1;
            unpack_f32x2(weights, p0, p1);
            pk[i] = pack2<BF16>(p0, p1);
          }
        };
        const bool fresh = step == first && h == 0;    // (no reference yet)
        if constexpr (kAhead) weigh();
        float mx[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) mx[u] = __uint_as_float(sv[u]);
#pragma unroll
        for (int i = 8; i < kMine; i += 16) {
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            if (i + 8 < kMine) mx[u] = max3(mx[u], __uint_as_float(sv[i + u]), __uint_as_float(sv[i + 8 + u]));
            else mx[u] = fmaxf(mx[u], __uint_as_float(sv[i + u]));
          }
        }
        const float m_new = kBiasProduct ? fmaxf(max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) + base, ref.m)
                                         : max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), max3(mx[6], mx[7], ref.m));
        const bool need = ref.asks(m_new, c, kRescaleThreshold) && m_new != -INFINITY;
        if (__any_sync(0xffffffffu, need)) {
          const float f = ref.move(m_new, c);
          if constexpr (kBiasProduct) ref.large = !(fabsf((m_new - base) * c) <= kFusedReference);
          if (!fresh) {
            // one P V at most is under way, the last half's: the one before was issued ahead of these scores
            if constexpr (!SPLIT) {
              ok = __all_sync(0xffffffffu, mbar_wait(&bar->pv_done[buf], h ^ 1, abort_word, 0x810));
              if (!ok) break;
              tc_fence_after_sync();
            }
#pragma unroll
            for (int cc = 0; cc < D; cc += 16) {
              uint32_t o[16];
              tmem_ld_x16_wait(o_col + buf * D + cc, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st_x16(o_col + buf * D + cc, o);
            }
            tmem_wait_st();
          }
          l *= f;
          if (kBiasProduct && __any_sync(0xffffffffu, ref.large && base != 0.f)) {
#pragma unroll
            for (int i = 0; i < kMine; ++i) sv[i] = __float_as_uint(__uint_as_float(sv[i]) + base);
            base = 0.f;
          }
          ref.subtract(sv);
          if constexpr (kAhead) weigh();
        }
        if constexpr (!kAhead) weigh();
        if constexpr (PAGED) {
          // the slots behind a sequence's end hold anything: their values become zeros, which their weights, zeros too, need
          if (h == 0 && (j + 1) * kKeys > s.keys) {      // (with two tiles both do this, and write the same)
            const int nv = 2 * (s.block0 + step - s.begin()) + 1, st = nv % kStages;
            ok = __all_sync(0xffffffffu, mbar_wait(&bar->kv_full[st], (nv / kStages) & 1, abort_word, 0x820));
            if (!ok) break;
            uint8_t* v = smem + LO::kOffKV + st * kTile;
            const int from = (s.keys - j * kKeys) * 8, pieces = kKeys * 8;      // 16-byte pieces of an atom
            for (int a = 0; a < kAtoms; ++a)
              for (int i = from + row; i < pieces; i += 128) *reinterpret_cast<uint4*>(v + a * (kKeys * 128) + i * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
          }
        }
        if constexpr (SPLIT) {
          // the keys of the other warps have no weight in this warp's copy of the rows
          uint32_t none[16] = {};
#pragma unroll
          for (int other = 1; other < 4; ++other) tmem_st_x16(s_col + ((quad + other) & 3) * 16, none);
          tmem_st_x16(s_col + quad * 16, pk);
        } else {
          tmem_st_x16(s_col + part0, *reinterpret_cast<uint32_t(*)[16]>(&pk[0]));
          tmem_st_x16(s_col + part0 + 16, *reinterpret_cast<uint32_t(*)[16]>(&pk[16]));
        }
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive_warp(&bar->p_full[buf][h], lane);
        float s0, s1;
        unpack_f32x2(add_f32x2(sum2[0], sum2[1]), s0, s1);
        l += s0 + s1;
       }
      }
      if (!ok) break;

      // The results of the item, or of the part of it.  Two tiles: a row's thread has all of it.  One tile: a row's two threads join the
      // accumulators, sum_b 2^(c (m_b - m)) O_b, half of the columns each.
      constexpr int kCols = NT == 2 ? D : D / 2;
      const int col0 = NT == 2 ? 0 : buf * kCols;
      bool has[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) has[b] = NT == 2 ? s.lo(b) < s.hi(b) : s.hi0 - s.lo0 > b;
      float f_mine = 1.0f, f_other = 0.f;
      if constexpr (NT == 1) {
        float2* both = sums + (segs & 1) * 256;
        both[buf * 128] = make_float2(ref.m, l);
        mbar_arrive_warp(&bar->sums_full, lane);
        ok = __all_sync(0xffffffffu, mbar_wait(&bar->sums_full, segs & 1, abort_word, 0x850));
        if (!ok) break;
        if constexpr (SPLIT) {
          const float2* all = both - row + lane;       // of the row's eight threads: buffer, copy
          float m = -INFINITY, sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (all[i * 32].y != 0.f) m = fmaxf(m, all[i * 32].x);
          auto factor = [&](float2 ml) { return ml.y == 0.f ? 0.f : ml.x == m ? 1.0f : ex2_approx((ml.x - m) * c); };
#pragma unroll
          for (int i = 0; i < 8; ++i) sum = fmaf(all[i * 32].y, factor(all[i * 32]), sum);
          f_mine = factor(make_float2(ref.m, l));
          f_other = factor(both[(buf ^ 1) * 128]);
          l = sum;
          ref.m = m;
        } else {
          const float2 other = both[(buf ^ 1) * 128];
          const float m = other.y == 0.f ? ref.m : l == 0.f ? other.x : fmaxf(ref.m, other.x);
          f_mine = ref.m == m ? 1.0f : l == 0.f ? 0.f : ex2_approx((ref.m - m) * c);
          f_other = other.y == 0.f ? 0.f : other.x == m ? 1.0f : ex2_approx((other.x - m) * c);
          l = l * f_mine + other.y * f_other;
          ref.m = m;
        }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if ((NT == 2 && b != buf) || !has[b]) continue;
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar->o_done[b], (done >> b) & 1, abort_word, 0x830));
        done ^= 1u << b;
      }
      if (!ok) break;
      tc_fence_after_sync();
      const float inv = s.part >= 0 ? 1.0f : l == 0.f ? 0.f : 1.0f / l;
      const size_t part_at = PAGED && s.part >= 0 ? ((static_cast<size_t>(blockIdx.x) * 2 + s.part) * NT + t) * (SPLIT ? 32 : kRows) + in_copy : 0;
      uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) +
                     2 * ((PAGED ? 0 : s.seq * p.out_batch) + (s.row0 + static_cast<long long>(token)) * p.out_token + head * p.out_head);
#pragma unroll
      for (int cc = 0; cc < kCols; cc += 16) {
        float o[16];
        {
          uint32_t x[16];
          const int b = NT == 2 ? buf : 0;
          if (has[b]) tmem_ld_x16_wait(o_col + b * D + col0 + cc, x);
          const float f = NT == 2 || buf == 0 ? f_mine : f_other;
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = has[b] ? __uint_as_float(x[i]) * f : 0.f;
        }
        if (NT == 1 && has[1]) {
          uint32_t x[16];
          tmem_ld_x16_wait(o_col + D + col0 + cc, x);
          const float f = buf == 0 ? f_other : f_mine;
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = fmaf(__uint_as_float(x[i]), f, o[i]);
        }
        if (cc + 16 == kCols) {
          tc_fence_before_sync();
#pragma unroll
          for (int b = 0; b < 2; ++b)
            if ((NT == 1 || b == buf) && has[b]) mbar_arrive_warp(&bar->o_free[b], lane);
        }
        if constexpr (SPLIT) {
          // the sum over the four copies: a warp takes four columns of a row each from the other warps of its buffer's half of the columns
          float* join = reinterpret_cast<float*>(smem + LO::kOffJoin) + (joins & 1) * (kSoftmaxWarps * 512) + buf * 2048;
#pragma unroll
          for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(join + (quad * 32 + lane) * 16 + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          mbar_arrive_warp(&bar->join_full, lane);
          ok = __all_sync(0xffffffffu, mbar_wait(&bar->join_full, joins & 1, abort_word, 0x860));
          if (!ok) break;
          ++joins;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int copy = 0; copy < 4; ++copy) {
            const float4 y = *reinterpret_cast<const float4*>(join + (copy * 32 + lane) * 16 + quad * 4);
            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
          }
          const int col = col0 + cc + quad * 4;
          if (valid && s.part >= 0) {
            if (l != 0.f) *reinterpret_cast<float4*>(p.part_o + part_at * D + col) = x;
          } else if (valid && col < p.d) {
            *reinterpret_cast<uint2*>(dst + 2 * col) =
                l == 0.f ? make_uint2(0, 0) : make_uint2(pack2<BF16>(x.x * inv, x.y * inv), pack2<BF16>(x.z * inv, x.w * inv));
          }
          continue;
        }
        if (!valid) continue;
        if (PAGED && s.part >= 0) {
          if (l != 0.f) {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<float4*>(p.part_o + part_at * D + col0 + cc + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
          continue;
        }
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
          uint32_t v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = l == 0.f ? 0u : pack2<BF16>(o[i + 2 * u] * inv, o[i + 2 * u + 1] * inv);
          if (col0 + cc + i < p.d) *reinterpret_cast<uint4*>(dst + 2 * (col0 + cc + i)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
      if (!ok) break;
      if (valid && (NT == 2 || buf == 0) && (!SPLIT || quad == 0)) {
        if (PAGED && s.part >= 0) p.part_ml[part_at] = make_float2(l == 0.f ? -INFINITY : ref.m, l);
        if (!PAGED && p.lse != nullptr)
          p.lse[(static_cast<size_t>(s.seq) * p.M + token) * p.heads + head] = l == 0.f ? -INFINITY : fmaf(ref.m * c, kLn2, logf(l));
      }
      if constexpr (PAGED) {
        if (s.part == 1 && threadIdx.x == 0) {
          // this CTA began the item: its parts end with the CTA whose share holds the item's last block
          const int share = blockIdx.x / p.lanes;
          const long long first_unit = static_cast<long long>(share) * bar->start.per_cta + s.at_unit;
          const int last_share = static_cast<int>((first_unit + s.units - 1) / bar->start.per_cta);
          p.parts[blockIdx.x] = {s.seq, s.kv_head, s.first_token, static_cast<int>(blockIdx.x) + (last_share - share) * p.lanes};
        }
      }
      mbar_arrive_warp(&bar->seg_empty[slot], lane);
    }
  }

  // After a wait has given up, TMA loads this CTA has armed may still be in flight; they complete within microseconds.
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

template <int D, bool BF16, int NT, bool PAGED, bool CAPPED, bool BIASED, bool SPLIT = false>
cudaError_t launch_one(const Params& p, int grid, cudaStream_t stream) {
  auto kern = masked_forward_kernel<D, BF16, NT, PAGED, CAPPED, BIASED, SPLIT>;
  static std::atomic<unsigned long long> configured{0};
  int dev = 0;
  cudaError_t e = current_device_checked(&dev);
  if (e != cudaSuccess) return e;
  if (!device_configured(configured, dev)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D, NT, SPLIT>::kBytes);
    if (e != cudaSuccess) return e;
    mark_device_configured(configured, dev);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Layout<D, NT, SPLIT>::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return launch_kernel(cfg, kern, p);
}

}  // namespace

namespace {
template <int D, bool BF16, bool PAGED, bool CAPPED, bool BIASED>
cudaError_t launch_tiles(const Params& p, int tiles, int grid, cudaStream_t stream) {
  if constexpr (PAGED) {
    if (tiles == 0) return launch_one<D, BF16, 1, PAGED, CAPPED, BIASED, true>(p, grid, stream);
  }
  return tiles == 2 ? launch_one<D, BF16, 2, PAGED, CAPPED, BIASED>(p, grid, stream) : launch_one<D, BF16, 1, PAGED, CAPPED, BIASED>(p, grid, stream);
}
}  // namespace

template <int D, bool BF16, bool PAGED>
cudaError_t launch_forward(const Params& p, int tiles, int grid, cudaStream_t stream) {
  if (p.cap_out != 0.f) return launch_tiles<D, BF16, PAGED, true, true>(p, tiles, grid, stream);      // (with slopes or without)
  return p.slopes != nullptr ? launch_tiles<D, BF16, PAGED, false, true>(p, tiles, grid, stream) : launch_tiles<D, BF16, PAGED, false, false>(p, tiles, grid, stream);
}

template cudaError_t launch_forward<(DITTO_MASKED_PART & 1) ? 128 : 64, (DITTO_MASKED_PART & 2) != 0, (DITTO_MASKED_PART & 4) != 0>(
    const Params&, int, int, cudaStream_t);

}  // namespace masked
}  // namespace ditto_b200
