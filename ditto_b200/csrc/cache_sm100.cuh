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

// Pools of pages that share one numbering (the keys and values of every layer): page i of a pool is `bytes` bytes at base + i * stride.
constexpr int kMaxPools = 256;
struct Pools {
  uint8_t* base[kMaxPools];
  long long stride;
  int count, pieces;          // pieces: 16-byte pieces of a page
};

// The tables of a cache: table [sequences, cols] of page ids (-1: none), lengths [sequences], references [pages] (how many entries of the
// table name a page; 0: free).
struct Tables {
  int *table, *lengths, *references;
  long long stride;
  int sequences, cols, page, pages;
  int* status;
};
// What the copy's launch does beside it; null pointers: nothing.  A fork (parents): the rows and lengths of the children and the references of
// their pages.  A compaction (renamed): the table with the pages' new names.
struct TableJob {
  Tables tables;
  const int *parents, *children, *target;
  const int* renamed;
  int* new_table;
  long long new_stride;
};

// Page copies target[i] <- source[i]; n is *n_device where that is not null.  A pair with a negative id is none.
struct CopyParams {
  Pools pools;
  const int *source, *target, *n_device;
  int n, pages;
  int* status;
  TableJob job;
};
cudaError_t launch_copy(const CopyParams& p, int sms, cudaStream_t stream);

cudaError_t launch_free(const Tables& t, const int* sequences, int n, cudaStream_t stream);
// lengths[b] += counts[b]; new pages are the lowest free ones, in the order of the sequences.  scratch: [sequences + 1].
cudaError_t launch_reserve(const Tables& t, const int* counts, int* scratch, cudaStream_t stream);
// Children take over their parents' full pages and get the lowest free pages for a copy of the last, in the order of the pairs: the page
// copies that remain to be made, source / target [n] and count, and with them the job of a fork; list [n]: scratch.
cudaError_t launch_fork(const Tables& t, const int* parents, const int* children, int n, int* source, int* target, int* list, int* count,
                        cudaStream_t stream);
// The live pages move to the front: new_references (which may be the old ones) from those of t; the page copies that remain to be made,
// source / target [pages] and count, and with them the job of a compaction, renamed [pages].
cudaError_t launch_compact(const Tables& t, int* new_references, int* renamed, int* source, int* target, int* count, cudaStream_t stream);

}  // namespace cache
}  // namespace ditto_b200
