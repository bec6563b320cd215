// Attention whose scores are capped, biased by distance and masked (dense, with gradients, and over a paged cache): what its kernels
// and the code that plans and launches them share.
//
// Query heads that share a key head are rows of one tile: row r of a tile is token r / group, head r % group of its key head, so that
// a tile of 128 rows covers 128 / group tokens whatever the number of heads, and a single token's heads cost one tile, not one each.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "sm100_ptx.cuh"

namespace ditto_b200 {
namespace masked {

constexpr int kRows = 128;        // rows of a query tile
constexpr int kKeys = 128;        // keys of a block

// Documents of a block of 128 keys: smallest and largest id that is not negative (an empty range where there is none).
struct KeyBlock {
  int least, most;
};

// An item that a CTA begins and does not end (split over several CTAs): what the combining kernel needs to find its parts.
struct PartDesc {
  int seq, kv_head, first_token;   // token inside the sequence of the item's first row
  int last_cta;                    // the part before is slot 1 of this CTA, then slot 0 of each up to this one; below 0: none
};

struct Params {
  CUtensorMap map_q;          // (d, heads, tokens, batch), box 64 x group x tokens of a tile x 1
  CUtensorMap map_k, map_v;   // (d, keys, kv heads, batch or pages), box 64 x min(128, page) x 1 x 1
  void* out;
  float* lse;                 // [batch, M, heads], may be null
  long long out_batch, out_token, out_head;    // strides in elements
  int batch, M, L;            // (paged: batch sequences; M is the number of tokens in all, L the table's reach in keys)
  int heads, kv_heads, group, tile_tokens, d;
  int tiles;                  // tiles of a batch entry (dense)
  int items;                  // batch x kv heads x groups of tiles (dense)
  int causal;
  float c;                    // factor of a score in the exponent of 2: scale log2(e), or 1 where cap or bias have applied it
  float cap_in, cap_out;      // scale / cap, and cap log2(e); cap_out 0: no cap
  float score_log2;           // scale log2(e)
  // forward, slopes without a cap: a slope times bias_unit is in the units of the scores times bias_factor.  bias_product: the scores' product
  // brings the bias of rows whose keys are all at or in front of them.
  float bias_unit, bias_factor;
  int bias_product;
  const float* slopes;        // [heads] or null
  const int* prefix;          // [batch] or null
  const int* documents;       // [batch, L] or null
  const int2* runs;           // [batch, L]: where the position's document begins and ends; (0, 0) of a negative one
  const int* mixed;           // [batch]: 1 where ids come in another order than rising, so that runs say nothing and ids are compared
  const int2* hulls;          // [batch, tiles]: first block and the one behind the last that the tile's documents reach
  // paged
  const int* table;
  const int* lengths;
  const int* starts;          // [batch + 1], or null: a token a sequence
  long long table_stride;
  int page, pages;
  int whole;                  // single tokens: CTA x has items x, x + grid, ... whole instead of a share of all blocks
  int lanes;                  // key heads that are worked on side by side: CTA x has heads x % lanes, + lanes, ... of its share of the blocks
  float* part_o;              // [CTA][2][tiles of an item x 128][D]
  float2* part_ml;            // [CTA][2][tiles of an item x 128]: reference (in scores) and sum
  PartDesc* parts;            // [CTA]
  int* status;
};

// codes of the status word beside those of expired waits: a page id out of range that a kernel passed over, too few free pages
constexpr int kBadPage = 0x10001, kNoPages = 0x10002;

// Blocks [lo, hi) of the keys of each tile of an item.
template <int NT>
struct Segment {
  int seq, kv_head, first_token;   // first token of tile 0, inside the sequence
  int tokens, keys;                // of the sequence
  int row0;                        // its first token's row in the tensors
  int prefix;
  int lo0, hi0, lo1, hi1;          // (scalars and not arrays: an index that is not known at compile time puts those into local memory)
  int part;                        // -1: the whole item; 0 or 1: the slot this part of it goes to
  int units, at_unit;              // paged: blocks of the whole item; blocks that this CTA has had before
  int block0;                      // K/V blocks that the CTA has loaded before
  int valid;                       // 0: there are no more

  __device__ __forceinline__ int lo(int t) const { return NT == 1 || t == 0 ? lo0 : lo1; }
  __device__ __forceinline__ int hi(int t) const { return NT == 1 || t == 0 ? hi0 : hi1; }
  // Blocks in the order in which they are taken: step i takes block i, or, from the last to the first, block begin + end - 1 - i.
  template <bool BACK>
  __device__ __forceinline__ int block(int i) const { return BACK ? begin() + end() - 1 - i : i; }
  template <bool BACK>
  __device__ __forceinline__ int first_step(int t) const { return BACK ? begin() + end() - hi(t) : lo(t); }
  template <bool BACK>
  __device__ __forceinline__ int last_step(int t) const { return BACK ? begin() + end() - lo(t) : hi(t); }
  __device__ __forceinline__ void set(int t, int lo, int hi) {
    if (t == 0) lo0 = lo, hi0 = hi;
    else lo1 = lo, hi1 = hi;
  }
  __device__ __forceinline__ void clear() { lo0 = hi0 = lo1 = hi1 = 0; }
  __device__ __forceinline__ bool used(int t, int j) const { return j >= lo(t) && j < hi(t); }
  __device__ __forceinline__ int begin() const { return NT == 1 || hi1 <= lo1 ? lo0 : hi0 <= lo0 ? lo1 : min(lo0, lo1); }
  __device__ __forceinline__ int end() const { return NT == 1 || hi1 <= lo1 ? hi0 : hi0 <= lo0 ? hi1 : max(hi0, hi1); }
};

// Keys that a query at `pos` sees without regard to documents: all below the answer.
__device__ __forceinline__ int visible_keys(int pos, int keys, int causal, int prefix) {
  const int e = causal ? max(pos + 1, prefix) : keys;
  return max(0, min(e, keys));
}

// Dense items, those with the most blocks first (causal: the last tiles), dealt out forwards and backwards in turn.
template <int NT>
struct DenseWalker {
  int round;
  __device__ __forceinline__ explicit DenseWalker() : round(0) {}
  template <class P>
  __device__ __forceinline__ bool next(const P& p, Segment<NT>& s) {
    const int grid = gridDim.x, at = round * grid + ((round & 1) ? grid - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x));
    ++round;
    if (round * grid - grid >= p.items) return false;
    if (at >= p.items) {                     // the last round's tail: an item of nothing
      s.tokens = 0, s.keys = 0, s.seq = -1;
      s.clear();
      return true;
    }
    const int heads_all = p.batch * p.kv_heads, per = p.items / heads_all;
    const int pair = per - 1 - at / heads_all, bh = at % heads_all;
    s.seq = bh / p.kv_heads;
    s.kv_head = bh % p.kv_heads;
    s.first_token = pair * NT * p.tile_tokens;
    s.tokens = p.M;
    s.keys = p.L;
    s.row0 = 0;
    s.prefix = p.prefix != nullptr ? p.prefix[s.seq] : 0;
    s.part = -1;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int tile = pair * NT + t;
      if (t == 0) s.clear();
      if (tile < p.tiles) {
        if (p.documents != nullptr) {
          const int2 h = p.hulls[static_cast<size_t>(s.seq) * p.tiles + tile];
          s.set(t, h.x, h.y);
        } else {
          const int last = min((tile + 1) * p.tile_tokens, p.M) - 1 + p.L - p.M;
          s.set(t, 0, (visible_keys(last, p.L, p.causal, s.prefix) + kKeys - 1) / kKeys);
        }
      }
    }
    return true;
  }
};

// Sequences of a paged cache.
struct Sequence {
  int row0, tokens, keys, prefix;
  __device__ __forceinline__ void load(const Params& p, int b) {
    row0 = b;
    tokens = 1;
    if (p.starts != nullptr) {
      row0 = max(0, min(p.starts[b], p.M));
      tokens = max(0, min(p.starts[b + 1], p.M) - row0);
    }
    keys = max(0, min(p.lengths[b], p.L));
    prefix = p.prefix != nullptr ? p.prefix[b] : 0;
  }
  // Blocks of the item of NT tiles that begins at token `first`; at least one, so that rows without keys are written too.
  template <int NT>
  __device__ __forceinline__ int units(const Params& p, int first) const {
    const int last = min(first + NT * p.tile_tokens, tokens) - 1 + keys - tokens;
    return max(1, (visible_keys(last, keys, p.causal, prefix) + kKeys - 1) / kKeys);
  }
  // ... of all items of one key head.
  template <int NT>
  __device__ __forceinline__ int units_of_head(const Params& p) const {
    int sum = 0;
    for (int first = 0; first < tokens; first += NT * p.tile_tokens) sum += units<NT>(p, first);
    return sum;
  }
};

// Where a CTA begins in the order (sequence, key head of its lane, tiles, block) of its lane's blocks, and how many it has; per_cta is everybody's
// share.  kv_head counts the heads of the lane.
struct PagedStart {
  int seq, kv_head, first_token, block, left, per_cta;
};

template <int NT>
struct PagedWalker {
  PagedStart at;
  int done;                    // blocks of this CTA so far
  Sequence q;
  __device__ __forceinline__ explicit PagedWalker(const PagedStart& s) : at(s), done(0) {}
  __device__ __forceinline__ bool next(const Params& p, Segment<NT>& s) {
    if (p.whole) {
      const int item = static_cast<int>(blockIdx.x) + at.left;       // (left counts up by the grid here)
      if (item >= p.batch * p.kv_heads) return false;
      at.left += gridDim.x;
      s.seq = item / p.kv_heads, s.kv_head = item % p.kv_heads;
      q.load(p, s.seq);
      s.first_token = 0, s.tokens = q.tokens, s.keys = q.keys, s.row0 = q.row0, s.prefix = q.prefix;
      s.part = -1, s.at_unit = 0;
      s.units = q.units<NT>(p, 0);
      s.clear();
      s.set(0, 0, (visible_keys(q.keys - 1, q.keys, p.causal, q.prefix) + kKeys - 1) / kKeys);
      return true;
    }
    if (at.left <= 0) return false;
    q.load(p, at.seq);
    while (at.first_token >= q.tokens) {        // the next key head, the next sequence with tokens
      at.first_token = 0;
      if (q.tokens == 0 || ++at.kv_head == p.kv_heads / p.lanes) {
        at.kv_head = 0;
        if (++at.seq >= p.batch) return false;
        q.load(p, at.seq);
      }
    }
    const int units = q.units<NT>(p, at.first_token), take = min(at.left, units - at.block);
    s.seq = at.seq;
    s.kv_head = at.kv_head * p.lanes + static_cast<int>(blockIdx.x) % p.lanes;
    s.first_token = at.first_token;
    s.tokens = q.tokens;
    s.keys = q.keys;
    s.row0 = q.row0;
    s.prefix = q.prefix;
    s.part = at.block > 0 ? 0 : take < units ? 1 : -1;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int first = at.first_token + t * p.tile_tokens;
      s.set(t, at.block, at.block);
      if (first < q.tokens) {
        const int last = min(first + p.tile_tokens, q.tokens) - 1 + q.keys - q.tokens;
        s.set(t, at.block, min(at.block + take, (visible_keys(last, q.keys, p.causal, q.prefix) + kKeys - 1) / kKeys));
      }
    }
    s.units = units;
    s.at_unit = done;
    at.left -= take;
    done += take;
    at.block += take;
    if (at.block == units) {
      at.block = 0;
      at.first_token += NT * p.tile_tokens;
    }
    return true;
  }
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int u) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(u)
      : "memory");
}

// tanh(x) = 1 - 2 / (1 + e^2x), to about 1.5e-7 absolute.
__device__ __forceinline__ float tanh_of(float x) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * 2.8853900817779268f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return fmaf(-2.0f, r, 1.0f);
}

// s <- f tanh(k s) for a thread's scores; the whole warp together.  Scores that are small beside the cap, the usual ones, take
// tanh(x) = x q(x^2) on the multiply-add pipe: q of degree 3 for |x| <= 0.35, of degree 5 for |x| <= 3/4, least maximum relative errors
// (iteratively reweighted least squares) 4.1e-8 and 2.9e-8.  tanh_of has two instructions of the special-function unit in it, which the exponentials
// behind keep busy already: the forward pass of 16 heads of 8192 x 8192 x 128, causal, took 529 us with it alone, 459 with degree 5, and in
// its present form takes 373 (252 without a cap).
template <int N>
__device__ __forceinline__ void capped(uint32_t (&s)[N], float k, float f) {
  const uint64_t k2 = pack_f32x2(k, k);
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint64_t x = mul_f32x2(pack_f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), k2);
    float x0, x1;
    unpack_f32x2(x, x0, x1);
    s[i] = __float_as_uint(x0), s[i + 1] = __float_as_uint(x1);
    most = max3(most, fabsf(x0), fabsf(x1));
  }
  auto both = [&](float c) { return pack_f32x2(f * c, f * c); };
  if (__all_sync(0xffffffffu, most <= 0.35f)) {
    const uint64_t c0 = both(1.0f), c1 = both(-0x1.555394p-2f), c2 = both(0x1.106164p-3f), c3 = both(-0x1.929fdep-5f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint64_t x = pack_f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), z = mul_f32x2(x, x);
      uint64_t q = fma_f32x2(c3, z, c2);
      q = fma_f32x2(q, z, c1);
      q = fma_f32x2(q, z, c0);
      float y0, y1;
      unpack_f32x2(mul_f32x2(x, q), y0, y1);
      s[i] = __float_as_uint(y0), s[i + 1] = __float_as_uint(y1);
    }
  } else if (__all_sync(0xffffffffu, most <= 0.75f)) {
    const uint64_t c0 = both(1.0f), c1 = both(-0x1.5554a4p-2f), c2 = both(0x1.10ed66p-3f), c3 = both(-0x1.b5604ep-5f), c4 = both(0x1.423392p-6f),
                   c5 = both(-0x1.389a58p-8f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint64_t x = pack_f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), z = mul_f32x2(x, x);
      uint64_t q = fma_f32x2(c5, z, c4);
      q = fma_f32x2(q, z, c3);
      q = fma_f32x2(q, z, c2);
      q = fma_f32x2(q, z, c1);
      q = fma_f32x2(q, z, c0);
      float y0, y1;
      unpack_f32x2(mul_f32x2(x, q), y0, y1);
      s[i] = __float_as_uint(y0), s[i + 1] = __float_as_uint(y1);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __float_as_uint(f * tanh_of(__uint_as_float(s[i])));
  }
}

// s <- f s - slope |far - i| for scores of keys i = 0 .. N - 1 of a query `far` positions behind the first of them.  Where no key that the row
// sees lies behind it (`linear`) the bias is linear in i: two instructions of the multiply-add pipe for two scores, with eight multiples of the
// slope in registers (a multiple a score would have to be loaded as a constant, two instructions more).
template <int N>
__device__ __forceinline__ void biased(uint32_t (&s)[N], float f, float slope, float far, bool linear) {
  if (linear) {
    const uint64_t f2 = pack_f32x2(f, f);
    uint64_t near[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) near[u] = pack_f32x2(slope * static_cast<float>(2 * u), slope * static_cast<float>(2 * u + 1));
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const float base = slope * (static_cast<float>(i) - far);
      const uint64_t base2 = pack_f32x2(base, base);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float y0, y1;
        unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[i + 2 * u]), __uint_as_float(s[i + 2 * u + 1])), f2, add_f32x2(near[u], base2)), y0, y1);
        s[i + 2 * u] = __float_as_uint(y0), s[i + 2 * u + 1] = __float_as_uint(y1);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __float_as_uint(fmaf(__uint_as_float(s[i]), f, -slope * fabsf(far - static_cast<float>(i))));
  }
}

// The launch of an instance of the forward kernel; grid: CTAs.  tiles: query tiles of an item, 1 or 2.
template <int D, bool BF16, bool PAGED>
cudaError_t launch_forward(const Params& p, int tiles, int grid, cudaStream_t stream);

}  // namespace masked

}  // namespace ditto_b200
