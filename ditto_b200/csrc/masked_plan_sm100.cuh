// Launches around the masked attention kernels (masked_plan_sm100.cu).
#pragma once
#include "masked_sm100.cuh"

namespace ditto_b200 {
namespace masked {

// documents [batch, L], the last M positions of a row being the queries': where every position's document begins and ends, what every block
// of keys holds, the blocks that every tile of queries reaches and, where key_hulls is not null, the tiles that reach every block.
cudaError_t launch_document_plan(const int* documents, const int* prefix, int batch, int M, int L, int causal, int tile_tokens, int tiles,
                                 int2* runs, int* mixed, KeyBlock* key_blocks, int2* hulls, int2* key_hulls, cudaStream_t stream);
cudaError_t launch_sum_parts(const Params& p, int d, bool bf16, int tiles, int grid, cudaStream_t stream);
cudaError_t launch_forward_any(const Params& p, int d, bool bf16, bool paged, int tiles, int grid, cudaStream_t stream);

}  // namespace masked
}  // namespace ditto_b200
