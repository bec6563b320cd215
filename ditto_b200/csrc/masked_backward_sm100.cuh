// Gradients of masked attention: what the kernels (masked_backward_sm100.cu) and their caller share.
#pragma once
#include "masked_sm100.cuh"

namespace ditto_b200 {
namespace masked {

// What the gradient kernels need of the 128 rows of a query tile, in the order of its rows; rows that are none have lse +infinity, which
// makes their weights zeros.
struct TileRows {
  float lse[kRows];      // log2 of the sum of exponentials
  float delta[kRows];    // sum over d of grad_out times out
  int doc[kRows];
  float slope[kRows];    // -slopes[head] log2(e)
  float pos[kRows];      // position of the row's query
};
static_assert(sizeof(TileRows) == 2560, "a bulk copy of whole 16-byte pieces");

// An item (kv head of a batch entry, block of keys) that a CTA begins and another ends.
struct KeyPartDesc {
  int item, last_cta;
};

struct BackwardParams {
  CUtensorMap map_q, map_do;  // (d, heads, tokens, batch), box 64 x group x tokens of a tile x 1
  CUtensorMap map_k, map_v;   // (d, keys, kv heads, batch), box 64 x 128 x 1 x 1
  const void *o, *grad;       // out and its gradient, for delta
  const void* v;
  long long o_stride[3], g_stride[3], v_stride[3];      // batch, token, head; in elements
  const float* lse;           // [batch, M, heads]
  void *dq, *dk, *dv;         // contiguous
  TileRows* rows;             // [batch][kv heads][tiles]
  uint32_t* norms;            // largest squared norms of a row of grad_out and of v, as the bits of a float; fp16 only
  int batch, M, L, heads, kv_heads, group, tile_tokens, d, tiles, blocks;
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
