// C ABI of the masked attention operators and the paged cache: argument checking, tensor maps, scratch memory, launches.
#include <climits>
#include <cmath>
#include <cstring>

#include "../../include/ditto_b200.h"
#include "cache_sm100.cuh"
#include "host_util.cuh"
#include "masked_backward_sm100.cuh"
#include "masked_plan_sm100.cuh"

namespace {

using namespace ditto_b200;

constexpr float kLog2e = 1.4426950408889634f;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
size_t up256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// strides of a [.., .., .., head_dim] operand in elements: whole 16-byte pieces
bool strides_ok(const long long* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] <= 0 || s[i] % 8 || s[i] >= (1ll << 38)) return false;
  return true;
}

int map_4d(CUtensorMap* map, bool bf16, const void* base, uint64_t d, uint64_t n1, uint64_t n2, uint64_t n3, long long s1, long long s2,
           long long s3, uint32_t b1, uint32_t b2) {
  const uint64_t dims[4] = {d, n1, n2, n3};
  const uint64_t strides[3] = {static_cast<uint64_t>(s1) * 2, static_cast<uint64_t>(s2) * 2, static_cast<uint64_t>(s3) * 2};
  const uint32_t box[4] = {64, b1, b2, 1};
  return make_tensor_map(map, bf16, base, 4, dims, strides, box);
}

int sm_count(int* sms) {
  static std::atomic<int> known[kMaxDevices];
  int dev = 0;
  cudaError_t e = current_device_checked(&dev);
  if (e != cudaSuccess) return cuda_fail("current device", e);
  int n = known[dev].load(std::memory_order_acquire);
  if (n == 0) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_fail("multiprocessor count", e);
    known[dev].store(n, std::memory_order_release);
  }
  *sms = n;
  return DITTO_OK;
}

// What the score rules of a call make of the kernel's constants.
int set_rules(masked::Params& p, float scale, float cap, const float* slopes, const int* prefix, int causal) {
  if (!(scale > 0.f) || !std::isfinite(scale) || !(cap >= 0.f) || !std::isfinite(cap)) return DITTO_ERR_INVALID_ARG;
  if (causal != 0 && causal != 1) return DITTO_ERR_INVALID_ARG;
  if (prefix != nullptr && !causal) return DITTO_ERR_INVALID_ARG;
  p.causal = causal;
  p.slopes = slopes;
  p.prefix = prefix;
  p.score_log2 = scale * kLog2e;
  p.cap_in = cap > 0.f ? scale / cap : 0.f;
  p.cap_out = cap > 0.f ? cap * kLog2e : 0.f;
  p.c = cap > 0.f || slopes != nullptr ? 1.0f : p.score_log2;
  return DITTO_OK;
}

// The forward kernel's units for a bias without a cap.  Its product brings the bias in units of the raw scores, slope / scale: scales so far out
// that this could leave the range of fp32 keep the bias in units of the exponent.
void set_bias_units(masked::Params& p, float scale) {
  p.bias_unit = kLog2e, p.bias_factor = p.score_log2, p.bias_product = 0;
  if (p.slopes == nullptr || p.cap_out != 0.f || scale < 0x1p-20f || scale > 0x1p20f) return;
  p.bias_unit = 1.0f / scale, p.bias_factor = 1.0f, p.bias_product = 1;
  p.c = p.score_log2;
}

int check_heads(int heads, int kv_heads, int d, int dtype) {
  if (heads <= 0 || kv_heads <= 0 || d <= 0) return DITTO_ERR_INVALID_ARG;
  if (dtype != DITTO_DTYPE_FP16 && dtype != DITTO_DTYPE_BF16) return DITTO_ERR_UNSUPPORTED;
  if (heads % kv_heads || heads / kv_heads > 128 || d % 8 || d > 128) return DITTO_ERR_UNSUPPORTED;
  return DITTO_OK;
}

int check_masked(const ditto_b200_masked_args* a) {
  if (!a || !a->q || !a->k || !a->v || !a->out) return DITTO_ERR_INVALID_ARG;
  if (a->batch <= 0 || a->M <= 0 || a->L <= 0) return DITTO_ERR_INVALID_ARG;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out)) return DITTO_ERR_INVALID_ARG;
  if (!strides_ok(a->q_strides, 3) || !strides_ok(a->k_strides, 3) || !strides_ok(a->v_strides, 3) || !strides_ok(a->out_strides, 3))
    return DITTO_ERR_INVALID_ARG;
  if (a->documents != nullptr && a->M > a->L) return DITTO_ERR_INVALID_ARG;
  return check_heads(a->heads, a->kv_heads, a->head_dim, a->dtype);
}

struct MaskedScratch {
  size_t mixed, key_blocks, hulls, key_hulls;      // of the documents, behind their runs
  size_t rows, norms, part, parts;       // of the backward pass
  size_t bytes;
};
// Tokens of a query tile of the gradient kernels.
int backward_tokens(int group) { return group <= masked::kHalf ? 2 * (masked::kHalf / group) : 1; }

MaskedScratch masked_scratch(const ditto_b200_masked_args* a, bool backward, int sms) {
  MaskedScratch s = {};
  const int group = a->heads / a->kv_heads;
  const size_t blocks = (a->L + 127) / 128, tile_tokens = backward ? backward_tokens(group) : 128 / group, tiles = (a->M + tile_tokens - 1) / tile_tokens;
  if (a->documents != nullptr) {
    s.mixed = up256(static_cast<size_t>(a->batch) * a->L * sizeof(int2));
    s.key_blocks = s.mixed + up256(a->batch * sizeof(int));
    s.hulls = s.key_blocks + up256(a->batch * blocks * sizeof(masked::KeyBlock));
    s.key_hulls = s.hulls + up256(a->batch * tiles * sizeof(int2));
    s.bytes = s.key_hulls + (backward ? up256(a->batch * blocks * sizeof(int2)) : 0);
  }
  if (backward) {
    s.rows = s.bytes;
    s.norms = s.rows + up256(a->batch * a->kv_heads * tiles * 2 * sizeof(masked::HalfRows));
    s.part = s.norms + 256;
    s.parts = s.part + static_cast<size_t>(sms) * 2 * 2 * 128 * (a->head_dim <= 64 ? 64 : 128) * sizeof(float);
    s.bytes = s.parts + up256(sms * sizeof(masked::KeyPartDesc));
  }
  return s;
}

// Launches the documents' plan of a call into its scratch memory and notes in p where what it finds is.
cudaError_t plan_documents(masked::Params& p, const MaskedScratch& ws, uint8_t* base, bool backward, cudaStream_t stream) {
  auto* runs = reinterpret_cast<int2*>(base);
  auto* mixed = reinterpret_cast<int*>(base + ws.mixed);
  auto* hulls = reinterpret_cast<int2*>(base + ws.hulls);
  p.runs = runs, p.mixed = mixed, p.hulls = hulls;
  return masked::launch_document_plan(p.documents, p.prefix, p.batch, p.M, p.L, p.causal, p.tile_tokens, p.tiles, runs, mixed,
                                      reinterpret_cast<masked::KeyBlock*>(base + ws.key_blocks), hulls,
                                      backward ? reinterpret_cast<int2*>(base + ws.key_hulls) : nullptr, stream);
}

// Query tiles of an item: two where that still leaves an item for every SM, so that each block of keys is loaded once for both.
int tiles_of_item(long long tiles, long long heads, int sms) { return tiles >= 2 && heads * ((tiles + 1) / 2) >= sms ? 2 : 1; }

int fill_masked(masked::Params& p, const ditto_b200_masked_args* a) {
  std::memset(&p, 0, sizeof(p));
  int rc = set_rules(p, a->scale, a->cap, a->slopes, a->prefix, a->causal);
  if (rc) return rc;
  const bool bf16 = a->dtype == DITTO_DTYPE_BF16;
  p.batch = a->batch;
  p.M = a->M;
  p.L = a->L;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.group = a->heads / a->kv_heads;
  p.tile_tokens = 128 / p.group;
  p.tiles = (a->M + p.tile_tokens - 1) / p.tile_tokens;
  p.d = a->head_dim;
  p.documents = a->documents;
  p.out = a->out;
  p.lse = a->lse;
  p.out_batch = a->out_strides[0];
  p.out_token = a->out_strides[1];
  p.out_head = a->out_strides[2];
  rc = map_4d(&p.map_q, bf16, a->q, p.d, p.heads, p.M, p.batch, a->q_strides[2], a->q_strides[1], a->q_strides[0], p.group, p.tile_tokens);
  if (rc) return rc;
  rc = map_4d(&p.map_k, bf16, a->k, p.d, p.L, p.kv_heads, p.batch, a->k_strides[1], a->k_strides[2], a->k_strides[0], 128, 1);
  if (rc) return rc;
  return map_4d(&p.map_v, bf16, a->v, p.d, p.L, p.kv_heads, p.batch, a->v_strides[1], a->v_strides[2], a->v_strides[0], 128, 1);
}

// The CTAs of a paged call and the query tiles of its items.
struct PagedPlan {
  int grid, tiles, lanes, whole;
  size_t part_ml, parts, bytes;
};
int paged_plan(const ditto_b200_paged_args* a, PagedPlan* plan) {
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc) return rc;
  const int group = a->heads / a->kv_heads, d = a->head_dim <= 64 ? 64 : 128;
  // 0: single tokens whose heads fill a quarter of a tile at most, in four copies of a row's heads.  Else as many tiles as the sequences have on
  // average: a second tile an item only where most sequences fill one.
  const int tile_tokens = 128 / group;
  plan->tiles = a->starts == nullptr && group <= 32 ? 0 : a->starts != nullptr && static_cast<long long>(a->tokens) > static_cast<long long>(a->batch) * tile_tokens ? 2 : 1;
  const long long items = (a->starts != nullptr ? a->tokens / (tile_tokens * plan->tiles) + static_cast<long long>(a->batch) : a->batch) * a->kv_heads;
  const long long most = items * ((static_cast<long long>(a->table_cols) * a->page + 127) / 128);
  if (most > INT_MAX) return DITTO_ERR_UNSUPPORTED;      // (blocks are counted in 32 bits)
  // Two heads of the same keys at the same time: their rows lie next to each other.  64 ragged sequences of up to 16384 keys, 8 key heads of 64:
  // 425 us instead of 537, of 128: 363 instead of 365; four lanes 443 and 359, eight 450 and 364.
  plan->lanes = a->kv_heads % 2 == 0 && most > sms ? 2 : 1;
  plan->grid = static_cast<int>(most < sms ? most : sms / plan->lanes * plan->lanes);
  // Single tokens of short sequences: items whole, and so no parts to be summed (a launch less) and no shares to be found.  8 heads over 2 of 64, by the
  // table's reach of 2, 4, 8 and 16 blocks: one sequence 7.6, 9.8, 14.4 and 23.4 us instead of 11.8, 12.1, 13.7 and 16.1, 32 sequences 8.3, 10.5, 15.1 and 24.0
  // instead of 12.4, 16.0, 17.8 and 19.4, 200 sequences 16.8, 23.7, 38.5 and 64.6 instead of 26.9, 31.7, 38.4 and 53.2.
  constexpr long long kWholeBlocks = 6;
  plan->whole = plan->tiles == 0 && (static_cast<long long>(a->table_cols) * a->page + 127) / 128 <= kWholeBlocks;
  if (plan->whole) plan->grid = static_cast<int>(items < sms ? items : sms);
  const size_t rows = static_cast<size_t>(plan->grid) * 2 * (plan->tiles == 0 ? 32 : plan->tiles * 128);
  plan->part_ml = up256(rows * d * sizeof(float));
  plan->parts = plan->part_ml + up256(rows * sizeof(float2));
  plan->bytes = plan->parts + up256(plan->grid * sizeof(masked::PartDesc));
  return DITTO_OK;
}

int check_paged(const ditto_b200_paged_args* a) {
  if (!a || !a->q || !a->key_pages || !a->value_pages || !a->out || !a->table || !a->lengths) return DITTO_ERR_INVALID_ARG;
  if (a->tokens <= 0 || a->batch <= 0 || a->pages <= 0 || a->page <= 0 || a->table_cols <= 0 || a->table_stride <= 0) return DITTO_ERR_INVALID_ARG;
  if (a->starts == nullptr && a->tokens != a->batch) return DITTO_ERR_INVALID_ARG;
  if (!aligned16(a->q) || !aligned16(a->key_pages) || !aligned16(a->value_pages) || !aligned16(a->out)) return DITTO_ERR_INVALID_ARG;
  if (!strides_ok(a->q_strides, 2) || !strides_ok(a->out_strides, 2) || !strides_ok(a->key_strides, 3) || !strides_ok(a->value_strides, 3))
    return DITTO_ERR_INVALID_ARG;
  const bool page_ok = a->page % 128 == 0 || a->page == 16 || a->page == 32 || a->page == 64;
  if (!page_ok || static_cast<long long>(a->table_cols) * a->page > (1ll << 30)) return DITTO_ERR_UNSUPPORTED;
  return check_heads(a->heads, a->kv_heads, a->head_dim, a->dtype);
}

int check_pools(const ditto_b200_pools* p) {
  if (!p || !p->base || p->count <= 0 || p->pages <= 0 || p->page_bytes <= 0 || p->stride_bytes < p->page_bytes) return DITTO_ERR_INVALID_ARG;
  if (p->page_bytes % 16 || p->stride_bytes % 16 || p->page_bytes > (1ll << 32)) return DITTO_ERR_INVALID_ARG;
  for (int i = 0; i < p->count; ++i)
    if (!p->base[i] || !aligned16(p->base[i])) return DITTO_ERR_INVALID_ARG;
  return DITTO_OK;
}

int check_tables(const ditto_b200_tables* t, bool page_needed, int* status_word, cache::Tables* out) {
  if (!t || !t->table || !t->references) return DITTO_ERR_INVALID_ARG;
  if (t->sequences <= 0 || t->cols <= 0 || t->pages <= 0 || t->stride < t->cols || (page_needed && t->page <= 0)) return DITTO_ERR_INVALID_ARG;
  *out = {t->table, t->lengths, t->references, t->stride, t->sequences, t->cols, t->page, t->pages, status_word};
  return DITTO_OK;
}

int copy_pages(const ditto_b200_pools* pools, const int* source, const int* target, const int* n_device, int n, const cache::TableJob& job,
               int* status_word, cudaStream_t stream) {
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc) return rc;
  cache::CopyParams p;
  p.pools.stride = pools->stride_bytes;
  p.pools.pieces = static_cast<int>(pools->page_bytes / 16);
  p.source = source;
  p.target = target;
  p.n_device = n_device;
  p.n = n;
  p.pages = pools->pages;
  p.status = status_word;
  p.job = job;
  for (int first = 0; first < pools->count; first += cache::kMaxPools) {
    p.pools.count = pools->count - first < cache::kMaxPools ? pools->count - first : cache::kMaxPools;
    for (int i = 0; i < p.pools.count; ++i) p.pools.base[i] = static_cast<uint8_t*>(pools->base[first + i]);
    const cudaError_t e = cache::launch_copy(p, sms, stream);
    if (e != cudaSuccess) return cuda_fail("cache page copy launch", e);
    p.job = {};                                        // (once)
  }
  return DITTO_OK;
}

}  // namespace

extern "C" {

size_t ditto_b200_masked_workspace_bytes(const ditto_b200_masked_args* a, int backward) {
  int sms = 0;
  if (check_masked(a) || (backward && sm_count(&sms))) return 0;
  return masked_scratch(a, backward != 0, sms).bytes;
}

int ditto_b200_masked_attention(const ditto_b200_masked_args* a, void* workspace, size_t ws_bytes, int* status_word, void* stream) {
  int rc = check_masked(a);
  if (rc) return rc;
  masked::Params p;
  rc = fill_masked(p, a);
  if (rc) return rc;
  set_bias_units(p, a->scale);
  const MaskedScratch ws = masked_scratch(a, false, 0);
  if (ws.bytes > 0 && (workspace == nullptr || ws_bytes < ws.bytes)) return DITTO_ERR_WORKSPACE;
  if (ws.bytes > 0 && !aligned16(workspace)) return DITTO_ERR_INVALID_ARG;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long heads = static_cast<long long>(p.batch) * p.kv_heads;
  const int nt = tiles_of_item(p.tiles, heads, sms);
  const long long items = heads * ((p.tiles + nt - 1) / nt);
  if (items > 0x3fffffffLL) return DITTO_ERR_UNSUPPORTED;
  p.items = static_cast<int>(items);
  p.status = status_word;
  if (a->documents != nullptr) {
    uint8_t* base = static_cast<uint8_t*>(workspace);
    const cudaError_t e = plan_documents(p, ws, base, false, st);
    if (e != cudaSuccess) return cuda_fail("masked_attention plan", e);
  }
  const cudaError_t e = masked::launch_forward_any(p, p.d <= 64 ? 64 : 128, a->dtype == DITTO_DTYPE_BF16, false, nt,
                                                   static_cast<int>(items < sms ? items : sms), st);
  if (e != cudaSuccess) return cuda_fail("masked_attention launch", e);
  return DITTO_OK;
}

int ditto_b200_masked_attention_backward(const ditto_b200_masked_args* a, const void* grad_out, const long long* grad_strides, void* dq, void* dk,
                                         void* dv, void* workspace, size_t ws_bytes, int* status_word, void* stream) {
  int rc = check_masked(a);
  if (rc) return rc;
  if (!a->lse || !grad_out || !grad_strides || !dq || !dk || !dv) return DITTO_ERR_INVALID_ARG;
  if (!aligned16(grad_out) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) || !strides_ok(grad_strides, 3)) return DITTO_ERR_INVALID_ARG;
  masked::Params f;
  rc = fill_masked(f, a);
  if (rc) return rc;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc) return rc;
  const MaskedScratch ws = masked_scratch(a, true, sms);
  if (workspace == nullptr || ws_bytes < ws.bytes) return DITTO_ERR_WORKSPACE;
  if (!aligned16(workspace)) return DITTO_ERR_INVALID_ARG;
  const bool bf16 = a->dtype == DITTO_DTYPE_BF16;
  masked::BackwardParams p;
  std::memset(&p, 0, sizeof(p));
  // halves of a tile: whole tokens, or half of one token's heads
  p.half_heads = f.group <= masked::kHalf ? f.group : (f.group + 1) / 2;
  p.head_step = f.group <= masked::kHalf ? 0 : p.half_heads;
  const int box_tokens = f.group <= masked::kHalf ? masked::kHalf / f.group : 1;
  p.half_tokens = f.group <= masked::kHalf ? box_tokens : 0;
  p.half_rows = p.half_heads * box_tokens;
  f.tile_tokens = backward_tokens(f.group);
  f.tiles = (f.M + f.tile_tokens - 1) / f.tile_tokens;
  rc = map_4d(&p.map_q, bf16, a->q, f.d, f.heads, f.M, f.batch, a->q_strides[2], a->q_strides[1], a->q_strides[0], p.half_heads, box_tokens);
  if (rc) return rc;
  rc = map_4d(&p.map_do, bf16, grad_out, f.d, f.heads, f.M, f.batch, grad_strides[2], grad_strides[1], grad_strides[0], p.half_heads, box_tokens);
  if (rc) return rc;
  rc = map_4d(&p.map_k, bf16, a->k, f.d, f.L, f.kv_heads, f.batch, a->k_strides[1], a->k_strides[2], a->k_strides[0], 64, 1);
  if (rc) return rc;
  rc = map_4d(&p.map_v, bf16, a->v, f.d, f.L, f.kv_heads, f.batch, a->v_strides[1], a->v_strides[2], a->v_strides[0], 64, 1);
  if (rc) return rc;
  p.o = a->out;
  p.grad = grad_out;
  p.v = a->v;
  for (int i = 0; i < 3; ++i) {
    p.o_stride[i] = a->out_strides[i];
    p.g_stride[i] = grad_strides[i];
    p.v_stride[i] = a->v_strides[i];
  }
  p.lse = a->lse;
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.batch = f.batch, p.M = f.M, p.L = f.L, p.heads = f.heads, p.kv_heads = f.kv_heads, p.group = f.group, p.tile_tokens = f.tile_tokens, p.d = f.d;
  p.tiles = f.tiles;
  p.blocks = (f.L + 127) / 128;
  const long long heads = static_cast<long long>(p.batch) * p.kv_heads;
  if (heads * p.tiles > 0x3fffffffLL || heads * p.blocks * p.tiles > 0x3fffffffLL) return DITTO_ERR_UNSUPPORTED;
  p.items = static_cast<int>(heads * p.tiles);
  p.causal = f.causal, p.c = f.c, p.cap_in = f.cap_in, p.cap_out = f.cap_out, p.score_log2 = f.score_log2, p.scale = a->scale;
  p.slopes = f.slopes, p.prefix = f.prefix, p.documents = f.documents;
  p.status = status_word;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  p.rows = reinterpret_cast<masked::HalfRows*>(base + ws.rows);
  p.norms = reinterpret_cast<uint32_t*>(base + ws.norms);
  p.part = reinterpret_cast<float*>(base + ws.part);
  p.parts = reinterpret_cast<masked::KeyPartDesc*>(base + ws.parts);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (a->documents != nullptr) {
    e = plan_documents(f, ws, base, true, st);
    p.runs = f.runs, p.mixed = f.mixed, p.hulls = f.hulls;
    p.key_hulls = reinterpret_cast<int2*>(base + ws.key_hulls);
  }
  if (e == cudaSuccess) {
    if (p.d <= 64)
      e = bf16 ? masked::launch_backward<64, true>(p, sms, st) : masked::launch_backward<64, false>(p, sms, st);
    else
      e = bf16 ? masked::launch_backward<128, true>(p, sms, st) : masked::launch_backward<128, false>(p, sms, st);
  }
  if (e != cudaSuccess) return cuda_fail("masked_attention_backward launch", e);
  return DITTO_OK;
}

size_t ditto_b200_paged_workspace_bytes(const ditto_b200_paged_args* a) {
  PagedPlan plan;
  if (check_paged(a) || paged_plan(a, &plan)) return 0;
  return plan.bytes;
}

int ditto_b200_paged_attention(const ditto_b200_paged_args* a, void* workspace, size_t ws_bytes, int* status_word, void* stream) {
  int rc = check_paged(a);
  if (rc) return rc;
  masked::Params p;
  std::memset(&p, 0, sizeof(p));
  rc = set_rules(p, a->scale, a->cap, a->slopes, a->prefix, 1);
  if (rc) return rc;
  set_bias_units(p, a->scale);
  PagedPlan plan;
  rc = paged_plan(a, &plan);
  if (rc) return rc;
  if (workspace == nullptr || ws_bytes < plan.bytes) return DITTO_ERR_WORKSPACE;
  if (!aligned16(workspace)) return DITTO_ERR_INVALID_ARG;
  const bool bf16 = a->dtype == DITTO_DTYPE_BF16;
  const int d = a->head_dim <= 64 ? 64 : 128;
  p.batch = a->batch;
  p.M = a->tokens;
  p.L = a->table_cols * a->page;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.group = a->heads / a->kv_heads;
  p.tile_tokens = plan.tiles == 0 ? 1 : 128 / p.group;
  p.d = a->head_dim;
  p.out = a->out;
  p.out_token = a->out_strides[0];
  p.out_head = a->out_strides[1];
  p.table = a->table;
  p.table_stride = a->table_stride;
  p.lengths = a->lengths;
  p.starts = a->starts;
  p.page = a->page;
  p.pages = a->pages;
  p.lanes = plan.lanes;
  p.whole = plan.whole;
  p.status = status_word;
  const long long q_all = a->q_strides[0] * static_cast<long long>(a->tokens);
  rc = map_4d(&p.map_q, bf16, a->q, p.d, p.heads, p.M, 1, a->q_strides[1], a->q_strides[0], q_all, p.group, p.tile_tokens);
  if (rc) return rc;
  const uint32_t rows = a->page < 128 ? a->page : 128;
  rc = map_4d(&p.map_k, bf16, a->key_pages, p.d, p.page, p.kv_heads, p.pages, a->key_strides[1], a->key_strides[2], a->key_strides[0], rows, 1);
  if (rc) return rc;
  rc = map_4d(&p.map_v, bf16, a->value_pages, p.d, p.page, p.kv_heads, p.pages, a->value_strides[1], a->value_strides[2], a->value_strides[0], rows, 1);
  if (rc) return rc;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  p.part_o = reinterpret_cast<float*>(base);
  p.part_ml = reinterpret_cast<float2*>(base + plan.part_ml);
  p.parts = reinterpret_cast<masked::PartDesc*>(base + plan.parts);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = masked::launch_forward_any(p, d, bf16, true, plan.tiles, plan.grid, st);
  if (e == cudaSuccess && !plan.whole) e = masked::launch_sum_parts(p, d, bf16, plan.tiles, plan.grid, st);
  if (e != cudaSuccess) return cuda_fail("paged_attention launch", e);
  return DITTO_OK;
}

int ditto_b200_cache_append(const ditto_b200_append_args* a, int* status_word, void* stream) {
  if (!a || !a->keys || !a->values || !a->key_pages || !a->value_pages || !a->table || !a->lengths) return DITTO_ERR_INVALID_ARG;
  if (a->tokens <= 0 || a->batch <= 0 || a->pages <= 0 || a->page <= 0 || a->table_cols <= 0 || a->table_stride <= 0 || a->kv_heads <= 0)
    return DITTO_ERR_INVALID_ARG;
  if (a->starts == nullptr && a->tokens != a->batch) return DITTO_ERR_INVALID_ARG;
  if (a->head_dim <= 0 || a->head_dim % 8) return DITTO_ERR_UNSUPPORTED;
  if (!aligned16(a->keys) || !aligned16(a->values) || !aligned16(a->key_pages) || !aligned16(a->value_pages)) return DITTO_ERR_INVALID_ARG;
  if (!strides_ok(a->k_strides, 2) || !strides_ok(a->v_strides, 2) || !strides_ok(a->key_strides, 3) || !strides_ok(a->value_strides, 3))
    return DITTO_ERR_INVALID_ARG;
  cache::AppendParams p = {};
  p.keys = static_cast<const uint8_t*>(a->keys);
  p.values = static_cast<const uint8_t*>(a->values);
  p.key_pages = static_cast<uint8_t*>(a->key_pages);
  p.value_pages = static_cast<uint8_t*>(a->value_pages);
  p.k_token = a->k_strides[0] * 2, p.k_head = a->k_strides[1] * 2;
  p.v_token = a->v_strides[0] * 2, p.v_head = a->v_strides[1] * 2;
  p.kp_page = a->key_strides[0] * 2, p.kp_slot = a->key_strides[1] * 2, p.kp_head = a->key_strides[2] * 2;
  p.vp_page = a->value_strides[0] * 2, p.vp_slot = a->value_strides[1] * 2, p.vp_head = a->value_strides[2] * 2;
  p.table = a->table;
  p.table_stride = a->table_stride;
  p.table_cols = a->table_cols;
  p.lengths = a->lengths;
  p.starts = a->starts;
  p.batch = a->batch;
  p.tokens = a->tokens;
  p.kv_heads = a->kv_heads;
  p.pieces = a->head_dim / 8;
  p.page = a->page;
  p.pages = a->pages;
  p.status = status_word;
  const cudaError_t e = cache::launch_append(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail("cache_append launch", e);
  return DITTO_OK;
}

int ditto_b200_cache_copy(const ditto_b200_pools* pools, const int* source, const int* target, int n, int* status_word, void* stream) {
  const int rc = check_pools(pools);
  if (rc) return rc;
  if (!source || !target || n <= 0) return DITTO_ERR_INVALID_ARG;
  return copy_pages(pools, source, target, nullptr, n, cache::TableJob{}, status_word, static_cast<cudaStream_t>(stream));
}

int ditto_b200_cache_free(const ditto_b200_tables* tables, const int* sequences, int n, int* status_word, void* stream) {
  cache::Tables t;
  const int rc = check_tables(tables, false, status_word, &t);
  if (rc) return rc;
  if (!t.lengths || !sequences || n <= 0) return DITTO_ERR_INVALID_ARG;
  const cudaError_t e = cache::launch_free(t, sequences, n, static_cast<cudaStream_t>(stream));
  return e != cudaSuccess ? cuda_fail("cache_free launch", e) : DITTO_OK;
}

size_t ditto_b200_cache_workspace_bytes(const ditto_b200_tables* t, int n) {
  if (!t || t->sequences < 0 || t->pages < 0 || n < 0) return 0;
  // reserve: a word a sequence and one more; fork: three a pair and one; compact: three a page and one
  const size_t words = 3 * (static_cast<size_t>(t->pages) > static_cast<size_t>(n) ? t->pages : n), seqs = t->sequences;
  return up256(((words > seqs ? words : seqs) + 1) * sizeof(int));
}

int ditto_b200_cache_reserve(const ditto_b200_tables* tables, const int* counts, void* workspace, size_t ws_bytes, int* status_word, void* stream) {
  cache::Tables t;
  const int rc = check_tables(tables, true, status_word, &t);
  if (rc) return rc;
  if (!t.lengths || !counts) return DITTO_ERR_INVALID_ARG;
  if (!workspace || ws_bytes < (static_cast<size_t>(t.sequences) + 1) * sizeof(int)) return DITTO_ERR_WORKSPACE;
  if (!aligned16(workspace)) return DITTO_ERR_INVALID_ARG;
  const cudaError_t e = cache::launch_reserve(t, counts, static_cast<int*>(workspace), static_cast<cudaStream_t>(stream));
  return e != cudaSuccess ? cuda_fail("cache_reserve launch", e) : DITTO_OK;
}

int ditto_b200_cache_fork(const ditto_b200_pools* pools, const ditto_b200_tables* tables, const int* parents, const int* children, int n,
                          void* workspace, size_t ws_bytes, int* status_word, void* stream) {
  cache::Tables t;
  int rc = check_tables(tables, true, status_word, &t);
  if (rc == DITTO_OK) rc = check_pools(pools);
  if (rc) return rc;
  if (!t.lengths || !parents || !children || n <= 0 || pools->pages != t.pages) return DITTO_ERR_INVALID_ARG;
  if (!workspace || ws_bytes < (3 * static_cast<size_t>(n) + 1) * sizeof(int)) return DITTO_ERR_WORKSPACE;
  if (!aligned16(workspace)) return DITTO_ERR_INVALID_ARG;
  int* count = static_cast<int*>(workspace);
  int *source = count + 1, *target = source + n, *list = target + n;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = cache::launch_fork(t, parents, children, n, source, target, list, count, st);
  if (e != cudaSuccess) return cuda_fail("cache_fork launch", e);
  cache::TableJob job = {};
  job.tables = t, job.parents = parents, job.children = children, job.target = target;
  return copy_pages(pools, source, target, count, n, job, status_word, st);
}

int ditto_b200_cache_compact(const ditto_b200_pools* pools, const ditto_b200_tables* tables, int* new_table, long long new_stride,
                             int* new_references, void* workspace, size_t ws_bytes, int* status_word, void* stream) {
  cache::Tables t;
  int rc = check_tables(tables, false, status_word, &t);
  if (rc == DITTO_OK) rc = check_pools(pools);
  if (rc) return rc;
  if (!new_table || !new_references || new_stride < t.cols || pools->pages != t.pages) return DITTO_ERR_INVALID_ARG;
  if (!workspace || ws_bytes < (3 * static_cast<size_t>(t.pages) + 1) * sizeof(int)) return DITTO_ERR_WORKSPACE;
  if (!aligned16(workspace)) return DITTO_ERR_INVALID_ARG;
  int* count = static_cast<int*>(workspace);
  int *source = count + 1, *target = source + t.pages, *renamed = target + t.pages;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = cache::launch_compact(t, new_references, renamed, source, target, count, st);
  if (e != cudaSuccess) return cuda_fail("cache_compact launch", e);
  cache::TableJob job = {};
  job.tables = t, job.renamed = renamed, job.new_table = new_table, job.new_stride = new_stride;
  return copy_pages(pools, source, target, count, t.pages, job, status_word, st);
}

}  // extern "C"
