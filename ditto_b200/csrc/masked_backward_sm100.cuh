// Gradients of masked attention: what the kernels (masked_backward_sm100.cu) and their caller share.
#pragma once
#include "masked_sm100.cuh"

namespace ditto_b200 {
namespace masked {

// The gradient kernels take a query tile in two halves of 64 rows, each of whole tokens (64 / group of them), or, where more than 64 heads
// share a key head, of half of one token's heads: the loads of a half go out as soon as the half of the tile before last is done with.
constexpr int kHalf = 64;

// What the gradient kernels need of a half's rows, in their order; rows that are none have -infinity for lse, which makes their weights zeros.
struct HalfRows {
  float lse[kHalf];      // -log2 of the sum of exponentials (negative: what is added to an exponent)
  float delta[kHalf];    // -sum over d of grad_out times out
  int doc[kHalf];
  float slope[kHalf];    // -slopes[head] log2(e)
  float pos[kHalf];      // position of the row's query
};
static_assert(sizeof(HalfRows) == 1280, "a bulk copy of whole 16-byte pieces");

// An item (kv head of a batch entry, block of keys) that a CTA begins and another ends.
struct KeyPartDesc {
  int item, last_cta;
};

struct BackwardParams {
  CUtensorMap map_q, map_do;  // (d, heads, tokens, batch), box 64 x half_heads x half's tokens x 1
  CUtensorMap map_k, map_v;   // (d, keys, kv heads, batch), box 64 x 64 x 1 x 1
  const void *o, *grad;       // out and its gradient, for delta
  const void* v;
  long long o_stride[3], g_stride[3], v_stride[3];      // batch, token, head; in elements
  const float* lse;           // [batch, M, heads]
  void *dq, *dk, *dv;         // contiguous
  HalfRows* rows;             // [batch][kv heads][tiles][2]
  uint32_t* norms;            // largest squared norms of a row of grad_out and of v, as the bits of a float; fp16 only
  int batch, M, L, heads, kv_heads, group, tile_tokens, d, tiles, blocks;
  // row r of half g of tile i: token i tile_tokens + g half_tokens + r / half_heads, head g head_step + r % half_heads; half_rows of them
  int half_tokens, half_heads, head_step, half_rows;
  int items;                  // query tiles in all
  int causal;
  float c, cap_in, cap_out, score_log2, scale;
  const float* slopes;
  const int* prefix;
  const int* documents;
  const int2* runs;           // with documents, as in the forward pass
  const int* mixed;
  const int2* hulls;          // [batch][tiles]
  const int2* key_hulls;      // [batch][blocks]
  float* part;                // [CTA][2][dK, dV][128][D]
  KeyPartDesc* parts;         // [CTA]
  int* status;
};

template <int D, bool BF16>
cudaError_t launch_backward(const BackwardParams& p, int sms, cudaStream_t stream);

}  // namespace masked
}  // namespace ditto_b200
