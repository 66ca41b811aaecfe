// api_paged.cu -- C ABI of the paged KV-cache operators.
#include <cmath>

#include "api_common.h"
#include "paged.cuh"

using namespace ctts;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

size_t type_size(int dtype) { return dtype == CTTS_BF16 ? 2 : 4; }

// a stride of `ld` elements that keeps rows of at least `width` elements apart and 16-byte aligned
bool stride_ok(int64_t ld, int64_t width, int dtype) {
  return ld >= width && ld <= (int64_t)1 << 36 && ld * (int64_t)type_size(dtype) % 16 == 0;
}

int check_pool(const ctts_paged_kv& kv) {
  CTTS_REQ(kv.dtype == CTTS_F32 || kv.dtype == CTTS_BF16, CTTS_ERR_ARG, "bad cache dtype");
  CTTS_REQ(kv.head_dim == 64 || kv.head_dim == 128, CTTS_ERR_ARG, "head_dim must be 64 or 128");
  CTTS_REQ(kv.n_pages > 0 && kv.n_kv_heads > 0 && kv.n_kv_heads <= 1024, CTTS_ERR_ARG, "bad page or KV head count");
  CTTS_REQ(kv.page_size >= 8 && kv.page_size <= 256 && (kv.page_size & (kv.page_size - 1)) == 0, CTTS_ERR_ARG,
           "page_size must be a power of two, 8 to 256");
  CTTS_REQ((int64_t)kv.n_pages * kv.page_size <= 0x7fffffff, CTTS_ERR_RANGE, "n_pages * page_size must fit 31 bits");
  // (a stride of a dimension of one is never used, but it has to be one that could be)
  CTTS_REQ(stride_ok(kv.page_stride, kv.head_dim, kv.dtype) && stride_ok(kv.token_stride, kv.head_dim, kv.dtype) &&
               stride_ok(kv.head_stride, kv.head_dim, kv.dtype),
           CTTS_ERR_ARG, "cache strides must be at least head_dim and multiples of 16 bytes");
  return CTTS_OK;
}

int check_pool_data(const ctts_paged_kv& kv) {
  CTTS_REQ(kv.k && kv.v, CTTS_ERR_ARG, "null cache");
  CTTS_REQ(aligned16(kv.k) && aligned16(kv.v), CTTS_ERR_ARG, "cache must be 16-byte aligned");
  return CTTS_OK;
}

int check_heads(const ctts_paged_kv& kv, int n_heads) {
  CTTS_REQ(n_heads > 0 && n_heads % kv.n_kv_heads == 0, CTTS_ERR_ARG, "n_heads must be a multiple of n_kv_heads");
  return CTTS_OK;
}

// What the workspace and the launch shape of an attention call follow from.
int check_attn(const ctts_paged_attn* p) {
  CTTS_REQ(p, CTTS_ERR_ARG, "null argument");
  int rc = check_pool(p->kv);
  if (rc == CTTS_OK) rc = check_heads(p->kv, p->n_heads);
  if (rc != CTTS_OK) return rc;
  CTTS_REQ(p->n_heads / p->kv.n_kv_heads <= 16, CTTS_ERR_ARG, "at most 16 query heads per KV head");
  CTTS_REQ(p->q_dtype == CTTS_F32 || (p->q_dtype == CTTS_BF16 && p->kv.dtype == CTTS_BF16), CTTS_ERR_ARG,
           "queries are float32, or bf16 over a bf16 cache");
  CTTS_REQ(p->batch > 0 && p->rows >= 0 && p->max_new >= 0 && p->max_pages > 0, CTTS_ERR_ARG, "bad size");
  CTTS_REQ(p->batch <= 1 << 30, CTTS_ERR_RANGE, "too many requests");  // (counted in strides of a block's threads)
  // (the last tile of keys, of 128 at most, ends below 2^31)
  CTTS_REQ((int64_t)p->max_pages * p->kv.page_size <= 0x7fffffff - 127, CTTS_ERR_RANGE, "max_pages * page_size must not exceed 2^31 - 128");
  CTTS_REQ((int64_t)p->rows * (p->n_heads / p->kv.n_kv_heads) <= 0x7fffffff, CTTS_ERR_RANGE, "too many rows");
  // what the heads of one row tile take of the line is divided in 32 bits (units of a tile: up to 5)
  CTTS_REQ(5 * ((int64_t)p->max_pages * p->kv.page_size / 64 + 3) * p->kv.n_kv_heads <= 0xffffffff, CTTS_ERR_RANGE,
           "too many keys and KV heads");
  return CTTS_OK;
}

}  // namespace

extern "C" int ctts_op_paged_plan(const ctts_paged_plan* p, void* stream) {
  CTTS_REQ(p && p->ctx_lens && p->new_lens && p->free_count && p->block_tables && p->free_pages && p->seq_lens &&
               p->cu_rows && p->state && (p->max_rows == 0 || (p->positions && p->slots)),
           CTTS_ERR_ARG, "null argument");
  CTTS_REQ(p->batch > 0 && p->max_pages > 0 && p->max_rows >= 0 && p->free_capacity >= 0 && p->table_ld >= p->max_pages,
           CTTS_ERR_ARG, "bad size");
  CTTS_REQ(p->batch <= kPlanMaxBatch, CTTS_ERR_RANGE, "at most 4096 requests in one plan");
  // (the kernel's counters go on by the grid's threads)
  CTTS_REQ(p->max_rows <= 1 << 30 && p->free_capacity <= 1 << 30, CTTS_ERR_RANGE, "at most 2^30 rows and free pages");
  CTTS_REQ(p->page_size >= 8 && p->page_size <= 256 && (p->page_size & (p->page_size - 1)) == 0, CTTS_ERR_ARG,
           "page_size must be a power of two, 8 to 256");
  CTTS_REQ((int64_t)p->max_pages * p->page_size <= 0x7fffffff, CTTS_ERR_RANGE, "max_pages * page_size must fit 31 bits");
  // CTAs read the inputs while others write the outputs
  const struct { const int* at; int64_t n; } in[] = {{p->ctx_lens, p->batch}, {p->new_lens, p->batch}, {p->free_count, 1}},
      out[] = {{p->seq_lens, p->batch}, {p->cu_rows, p->batch + 1}, {p->positions, p->max_rows}, {p->slots, p->max_rows}, {p->state, 4}};
  for (auto& i : in)
    for (auto& o : out)
      CTTS_REQ(o.n == 0 || i.at + i.n <= o.at || o.at + o.n <= i.at, CTTS_ERR_ARG, "an output overlaps an input");
  CTTS_CK(launch_paged_plan(*p, as_stream(stream, 0)));
  return CTTS_OK;
}

extern "C" int ctts_op_paged_append(const ctts_paged_append* p, void* stream) {
  CTTS_REQ(p, CTTS_ERR_ARG, "null argument");
  int rc = check_pool(p->kv);
  if (rc == CTTS_OK) rc = check_heads(p->kv, p->n_heads);
  if (rc != CTTS_OK) return rc;
  CTTS_REQ((p->x_dtype == CTTS_F32 || p->x_dtype == CTTS_BF16) && (p->q_dtype == CTTS_F32 || p->q_dtype == CTTS_BF16), CTTS_ERR_ARG,
           "bad dtype");
  CTTS_REQ(p->rows <= 1 << 30, CTTS_ERR_RANGE, "too many rows");
  CTTS_REQ(p->rows >= 0 && p->theta > 0.0 && std::isfinite(p->theta) && p->eps >= 0.0f, CTTS_ERR_ARG, "bad size, theta or eps");
  CTTS_REQ(!p->q_norm == !p->k_norm, CTTS_ERR_ARG, "q_norm and k_norm come together");
  const int64_t width = (int64_t)(p->n_heads + 2 * p->kv.n_kv_heads) * p->kv.head_dim;
  CTTS_REQ(width <= 1 << 24, CTTS_ERR_RANGE, "row too wide");
  CTTS_REQ(stride_ok(p->x_ld, width, p->x_dtype) && stride_ok(p->q_ld, (int64_t)p->n_heads * p->kv.head_dim, p->q_dtype), CTTS_ERR_ARG,
           "x_ld and q_ld must hold a row and be multiples of 16 bytes");
  if (p->rows == 0) return CTTS_OK;
  rc = check_pool_data(p->kv);
  if (rc != CTTS_OK) return rc;
  CTTS_REQ(p->x && p->q && p->positions && p->slots, CTTS_ERR_ARG, "null argument");
  CTTS_REQ(aligned16(p->x) && aligned16(p->q) && aligned16(p->q_norm) && aligned16(p->k_norm), CTTS_ERR_ARG,
           "x, q, q_norm and k_norm must be 16-byte aligned");
  CTTS_CK(launch_paged_append(*p, as_stream(stream, 0)));
  return CTTS_OK;
}

extern "C" int ctts_op_paged_attention_workspace(const ctts_paged_attn* p, size_t* bytes) {
  CTTS_REQ(bytes, CTTS_ERR_ARG, "null argument");
  const int rc = check_attn(p);
  if (rc != CTTS_OK) return rc;
  CTTS_REQ(paged_attn_plan(*p).ctas > 0, CTTS_ERR_CUDA, "no CUDA device");
  *bytes = paged_attn_ws_bytes(*p);
  return CTTS_OK;
}

extern "C" int ctts_op_paged_attention(const ctts_paged_attn* p, void* stream) {
  int rc = check_attn(p);
  if (rc != CTTS_OK) return rc;
  // (its factor to powers of two has to stay clear of zero and infinity, which make NaN of hidden scores)
  CTTS_REQ(p->scale >= 1e-20f && p->scale <= 1e20f, CTTS_ERR_ARG, "scale must lie between 1e-20 and 1e20");
  const int64_t width = (int64_t)p->n_heads * p->kv.head_dim;
  CTTS_REQ(stride_ok(p->q_ld, width, p->q_dtype) && stride_ok(p->out_ld, width, p->q_dtype) && p->table_ld >= p->max_pages, CTTS_ERR_ARG,
           "q_ld, out_ld and table_ld must hold a row (q_ld and out_ld in multiples of 16 bytes)");
  if (p->rows == 0 || p->max_new == 0) return CTTS_OK;
  rc = check_pool_data(p->kv);
  if (rc != CTTS_OK) return rc;
  CTTS_REQ(p->q && p->out && p->block_tables && p->cu_rows && p->seq_lens && p->workspace, CTTS_ERR_ARG, "null argument");
  CTTS_REQ(aligned16(p->q) && aligned16(p->out) && aligned16(p->workspace), CTTS_ERR_ARG, "q, out and workspace must be 16-byte aligned");
  const PagedAttnPlan pl = paged_attn_plan(*p);
  CTTS_REQ(pl.ctas > 0, CTTS_ERR_CUDA, "no CUDA device");
  CTTS_REQ(p->workspace_bytes >= pl.ws_bytes, CTTS_ERR_ARG, "workspace too small: " + std::to_string(pl.ws_bytes) + " bytes wanted");
  // the units of one CTA are counted in 31 bits (a tile is up to 5; a long item has 128 packed rows or more)
  const double group = p->n_heads / p->kv.n_kv_heads, tiles = (double)p->max_pages * p->kv.page_size / 64 + 3;
  CTTS_REQ(5 * tiles * p->kv.n_kv_heads * p->batch * (std::min(p->max_new, p->rows) * group / 128 + 1) <
               2147483647.0 * pl.ctas,
           CTTS_ERR_RANGE, "too many key tiles");
  CTTS_CK(launch_paged_attn(*p, as_stream(stream, 0)));
  return CTTS_OK;
}
