// Launches of the paged cache's kernels (cache_sm100.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ditto_b200 {
namespace cache {

// New tokens' rows to their places: token t of sequence b goes to position lengths[b] - (its tokens) + t.
struct AppendParams {
  const uint8_t *keys, *values;               // [tokens, kv heads, d], 16 bits an element
  uint8_t *key_pages, *value_pages;           // [pages, page, kv heads, d]
  long long k_token, k_head, v_token, v_head;                          // strides in bytes
  long long kp_page, kp_slot, kp_head, vp_page, vp_slot, vp_head;      // in bytes
  const int *table, *lengths, *starts;        // starts null: a token a sequence
  long long table_stride;
  int table_cols, batch, tokens, kv_heads, pieces;                     // 16-byte pieces of a head's row
  int page, pages;
  int* status;
};
cudaError_t launch_append(const AppendParams& p, cudaStream_t stream);

}  // namespace cache
}  // namespace ditto_b200
