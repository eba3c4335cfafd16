// extern "C" entry points of the paged-cache operators (declared in
// include/dequant_b200.h): argument checks, tensor maps, launches. Nothing
// here allocates device memory, synchronises or throws.
#include <cstdint>
#include <cstring>
#include <cuda_runtime.h>

#include "capi_checks.h"

namespace {

// The cache's description, checked; *pool is what the launchers take.
int check_pool(const dqg_paged_kv* kv, dqg::PagedPool* pool) {
  if (kv == nullptr) return api_fail(DQG_ERR_INVALID, "kv must not be null");
  int rc = check_ptr(kv->k, 16, "k_pages");
  if (rc) return rc;
  if ((rc = check_ptr(kv->v, 16, "v_pages")) != DQG_OK) return rc;
  if (kv->dtype != DQG_FP16 && kv->dtype != DQG_BF16)
    return api_fail(DQG_ERR_INVALID, "dtype must be DQG_FP16 or DQG_BF16, got %d", kv->dtype);
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return api_fail(DQG_ERR_UNSUPPORTED, "paged operators handle head_dim 64 and 128, got %lld",
                    (ll)kv->head_dim);
  const int64_t ps = kv->page_size;
  if (ps < 16 || ps > 256 || (ps & (ps - 1)))
    return api_fail(DQG_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256, got %lld", (ll)ps);
  if (kv->n_kv_heads < 1 || kv->n_kv_heads > 1024)
    return api_fail(DQG_ERR_INVALID, "n_kv_heads must be in [1, 1024], got %lld", (ll)kv->n_kv_heads);
  if (kv->n_pages < 1 || kv->n_pages > (int64_t(1) << 30))
    return api_fail(DQG_ERR_INVALID, "n_pages must be in [1, 2^30], got %lld", (ll)kv->n_pages);
  // A dimension of one element has no stride to speak of.
  const int64_t st[3] = {kv->n_pages > 1 ? kv->page_stride : kv->row_stride,
                         kv->n_kv_heads > 1 ? kv->head_stride : kv->row_stride, kv->row_stride};
  const char* names[3] = {"page", "head", "row"};
  for (int i = 0; i < 3; ++i)
    if (st[i] < 1 || st[i] % 8 || st[i] > (int64_t(1) << 38))
      return api_fail(DQG_ERR_INVALID, "the pools' %s stride must be a positive multiple of 8 elements, got %lld",
                      names[i], (ll)st[i]);
  if (kv->row_stride < kv->head_dim)
    return api_fail(DQG_ERR_INVALID, "the pools' rows overlap (row stride %lld)", (ll)kv->row_stride);
  pool->k = kv->k;
  pool->v = kv->v;
  pool->n_pages = kv->n_pages;
  pool->page_stride = st[0];
  pool->head_stride = st[1];
  pool->row_stride = st[2];
  pool->n_kv_heads = static_cast<int>(kv->n_kv_heads);
  pool->page_size = static_cast<int>(ps);
  pool->D = static_cast<int>(kv->head_dim);
  pool->bf16 = kv->dtype == DQG_BF16;
  return DQG_OK;
}

}  // namespace

extern "C" {

int dqg_rope_paged_append(const void* qkv, int64_t T, int64_t qkv_stride, int64_t n_q_heads,
                          const float* cos_table, const float* sin_table, int64_t n_positions,
                          int64_t rotary_dim, int interleaved, const int64_t* positions,
                          const int64_t* slots, const void* q_norm, const void* k_norm, float eps,
                          const dqg_paged_kv* kv, void* q_out, void* stream) {
  dqg::PagedPool pool;
  int rc = check_pool(kv, &pool);
  if (rc) return rc;
  if ((rc = check_heads(n_q_heads, pool.n_kv_heads)) != DQG_OK) return rc;
  if (T < 0 || T > (1 << 28)) return api_fail(DQG_ERR_INVALID, "T=%lld out of range", (ll)T);
  if (T == 0) return api_ok();
  const int64_t width = (n_q_heads + 2 * pool.n_kv_heads) * pool.D;
  if (qkv_stride < width || qkv_stride % 8)
    return api_fail(DQG_ERR_INVALID, "qkv's row stride must be a multiple of 8 and at least %lld, got %lld",
                    (ll)width, (ll)qkv_stride);
  if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > pool.D)
    return api_fail(DQG_ERR_INVALID, "rotary_dim must be even and in [2, head_dim], got %lld", (ll)rotary_dim);
  if (n_positions < 1)
    return api_fail(DQG_ERR_INVALID, "the cos/sin tables must hold at least one position");
  if ((q_norm == nullptr) != (k_norm == nullptr))
    return api_fail(DQG_ERR_INVALID, "q_norm and k_norm are given together or not at all");
  if (!(eps >= 0.f)) return api_fail(DQG_ERR_INVALID, "eps must be non-negative");
  const void* ptrs[8] = {qkv, cos_table, sin_table, positions, slots, q_out, q_norm, k_norm};
  const char* names[8] = {"qkv", "cos", "sin", "positions", "slots", "q_out", "q_norm", "k_norm"};
  const size_t align[8] = {16, 4, 4, 8, 8, 16, 16, 16};
  for (int i = 0; i < (q_norm ? 8 : 6); ++i)
    if ((rc = check_ptr(ptrs[i], align[i], names[i])) != DQG_OK) return rc;
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  dqg::AppendArgs a;
  a.qkv = qkv;
  a.qkv_stride = qkv_stride;
  a.cosv = cos_table;
  a.sinv = sin_table;
  a.positions = positions;
  a.slots = slots;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.q_out = q_out;
  a.n_positions = n_positions;
  a.T = static_cast<int>(T);
  a.hq = static_cast<int>(n_q_heads);
  a.rot = static_cast<int>(rotary_dim);
  a.eps = eps;
  a.interleaved = interleaved != 0;
  const cudaError_t e = dqg::launch_paged_append(pool, a, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(e, "rope_paged_append launch");
  return api_ok();
}

int dqg_paged_attention_workspace(int64_t n_seqs, int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                                  uint64_t* bytes) {
  return dqg_shared_prefix_workspace(n_seqs, n_q_heads, n_kv_heads, head_dim, 0, bytes);
}

int dqg_paged_attention(const void* q, int64_t q_stride_seq, int64_t q_stride_head, int64_t n_seqs,
                        int64_t n_q_heads, const dqg_paged_kv* kv, const int32_t* block_table,
                        int64_t table_width, int64_t table_stride, const int32_t* kv_lens, float scale,
                        void* out, void* workspace, uint64_t workspace_bytes, void* stream) {
  dqg::PagedPool pool;
  int rc = check_pool(kv, &pool);
  if (rc) return rc;
  if ((rc = check_heads(n_q_heads, pool.n_kv_heads)) != DQG_OK) return rc;
  if (n_seqs < 0 || n_seqs > (1 << 20))
    return api_fail(DQG_ERR_INVALID, "n_seqs=%lld out of range", (ll)n_seqs);
  if (n_seqs == 0) return api_ok();
  if ((rc = check_query(q, n_seqs, n_q_heads, q_stride_seq, q_stride_head, pool.D)) != DQG_OK) return rc;
  if ((rc = check_table(block_table, table_width, table_stride, "block_table")) != DQG_OK) return rc;
  if ((rc = check_ptr(kv_lens, 4, "kv_lens")) != DQG_OK) return rc;
  if ((rc = check_ptr(out, 16, "out")) != DQG_OK) return rc;
  if ((rc = check_scale(scale)) != DQG_OK) return rc;
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  if ((rc = check_workspace(workspace, workspace_bytes, dqg::paged_decode_workspace(static_cast<int>(n_seqs), static_cast<int>(n_q_heads), pool.n_kv_heads,
                                                    pool.D, 0, sms))) != DQG_OK)
    return rc;
  CUtensorMap kmap, vmap;
  if ((rc = pool_maps(pool, dqg::paged_decode_box_rows(pool.page_size), &kmap, &vmap)) != DQG_OK) return rc;
  dqg::DecodeArgs a;
  std::memset(&a, 0, sizeof(a));
  a.q = q;
  a.q_stride_seq = q_stride_seq;
  a.q_stride_head = q_stride_head;
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_width = static_cast<int>(table_width);
  a.lens = kv_lens;
  a.out = out;
  a.workspace = workspace;
  a.B = static_cast<int>(n_seqs);
  a.hq = static_cast<int>(n_q_heads);
  a.scale_log2 = static_cast<float>(scale * kLog2e);
  const cudaError_t e = dqg::launch_paged_decode(pool, kmap, vmap, a, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(e, "paged_attention launch");
  return api_ok();
}

int dqg_prompt_attention_workspace(int64_t head_dim, uint64_t* bytes) {
  if (bytes == nullptr) return api_fail(DQG_ERR_INVALID, "bytes must not be null");
  if (head_dim != 64 && head_dim != 128)
    return api_fail(DQG_ERR_UNSUPPORTED, "paged operators handle head_dim 64 and 128, got %lld", (ll)head_dim);
  int dev = 0, sms = 0;
  const int rc = current(&dev, &sms);
  if (rc) return rc;
  *bytes = dqg::prompt_workspace(static_cast<int>(head_dim), sms);
  return api_ok();
}

int dqg_prompt_attention(const void* q, int64_t q_stride_row, int64_t q_stride_head, int64_t T,
                         int64_t n_q_heads, const dqg_paged_kv* kv, const int32_t* block_table,
                         int64_t table_width, int64_t table_stride, const int32_t* q_starts,
                         const int32_t* kv_lens, int64_t n_seqs, int causal, float scale, void* out,
                         void* workspace, uint64_t workspace_bytes, void* stream) {
  dqg::PagedPool pool;
  int rc = check_pool(kv, &pool);
  if (rc) return rc;
  if ((rc = check_heads(n_q_heads, pool.n_kv_heads)) != DQG_OK) return rc;
  if (T < 0 || T > (1 << 28)) return api_fail(DQG_ERR_INVALID, "T=%lld out of range", (ll)T);
  if (n_seqs < 0 || n_seqs > (1 << 24))
    return api_fail(DQG_ERR_INVALID, "n_seqs=%lld out of range", (ll)n_seqs);
  if (T == 0 || n_seqs == 0) return api_ok();
  if ((rc = check_query(q, T, n_q_heads, q_stride_row, q_stride_head, pool.D)) != DQG_OK) return rc;
  if ((rc = check_table(block_table, table_width, table_stride, "block_table")) != DQG_OK) return rc;
  if ((rc = check_ptr(q_starts, 4, "q_starts")) != DQG_OK) return rc;
  if ((rc = check_ptr(kv_lens, 4, "kv_lens")) != DQG_OK) return rc;
  if ((rc = check_ptr(out, 16, "out")) != DQG_OK) return rc;
  if ((rc = check_scale(scale)) != DQG_OK) return rc;
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  if ((rc = check_workspace(workspace, workspace_bytes, dqg::prompt_workspace(pool.D, sms))) != DQG_OK)
    return rc;
  CUtensorMap qmap, kmap, vmap;
  if ((rc = query_map(q, pool, T, n_q_heads, q_stride_row, q_stride_head, &qmap)) != DQG_OK) return rc;
  if ((rc = pool_maps(pool, dqg::prompt_box_rows(pool.page_size), &kmap, &vmap)) != DQG_OK) return rc;
  dqg::PromptArgs a;
  std::memset(&a, 0, sizeof(a));
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_width = static_cast<int>(table_width);
  a.q_starts = q_starts;
  a.kv_lens = kv_lens;
  a.out = out;
  a.workspace = workspace;
  a.B = static_cast<int>(n_seqs);
  a.T = static_cast<int>(T);
  a.hq = static_cast<int>(n_q_heads);
  a.causal = causal != 0;
  a.scale_log2 = static_cast<float>(scale * kLog2e);
  const cudaError_t e = dqg::launch_prompt(pool, qmap, kmap, vmap, a, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(e, "prompt_attention launch");
  return api_ok();
}

int dqg_shared_prefix_workspace(int64_t n_seqs, int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                                int64_t prefix_len, uint64_t* bytes) {
  if (bytes == nullptr) return api_fail(DQG_ERR_INVALID, "bytes must not be null");
  if (head_dim != 64 && head_dim != 128)
    return api_fail(DQG_ERR_UNSUPPORTED, "paged operators handle head_dim 64 and 128, got %lld", (ll)head_dim);
  if (n_kv_heads < 1 || n_kv_heads > 1024)
    return api_fail(DQG_ERR_INVALID, "n_kv_heads must be in [1, 1024], got %lld", (ll)n_kv_heads);
  int rc = check_heads(n_q_heads, static_cast<int>(n_kv_heads));
  if (rc) return rc;
  if (n_seqs < 0 || n_seqs > (1 << 20))
    return api_fail(DQG_ERR_INVALID, "n_seqs=%lld out of range", (ll)n_seqs);
  if (prefix_len < 0 || prefix_len > (1 << 30))
    return api_fail(DQG_ERR_INVALID, "prefix_len=%lld out of range", (ll)prefix_len);
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  const bool pieces = prefix_len > 0 && n_seqs > 0 &&
                      !dqg::prefix_streamed(static_cast<int>(n_seqs), static_cast<int>(n_q_heads),
                                            static_cast<int>(n_kv_heads), static_cast<int>(head_dim),
                                            static_cast<int>(prefix_len));
  *bytes = dqg::paged_decode_workspace(static_cast<int>(n_seqs), static_cast<int>(n_q_heads),
                                       static_cast<int>(n_kv_heads), static_cast<int>(head_dim),
                                       static_cast<int>(prefix_len), sms);
  if (pieces)
    *bytes += dqg::prefix_workspace(static_cast<int>(n_seqs), static_cast<int>(n_q_heads),
                                    static_cast<int>(n_kv_heads), static_cast<int>(head_dim),
                                    static_cast<int>(prefix_len), sms);
  return api_ok();
}

}  // extern "C"

namespace {
int shared_prefix(const void* q, int64_t q_stride_seq, int64_t q_stride_head, int64_t n_seqs,
                  int64_t n_q_heads, const dqg_paged_kv* kv, const int32_t* prefix_table,
                  int64_t prefix_pages, int64_t prefix_len, const int32_t* block_table, int64_t table_width,
                  int64_t table_stride, const int32_t* kv_lens, float scale, void* out, void* workspace,
                  uint64_t workspace_bytes, uint32_t starved, uint64_t wait_ns, void* stream) {
  dqg::PagedPool pool;
  int rc = check_pool(kv, &pool);
  if (rc) return rc;
  uint64_t need = 0;
  rc = dqg_shared_prefix_workspace(n_seqs, n_q_heads, pool.n_kv_heads, pool.D, prefix_len, &need);
  if (rc) return rc;
  if (n_seqs == 0) return api_ok();
  if ((rc = check_query(q, n_seqs, n_q_heads, q_stride_seq, q_stride_head, pool.D)) != DQG_OK) return rc;
  if ((rc = check_table(block_table, table_width, table_stride, "block_table")) != DQG_OK) return rc;
  if (prefix_len > 0) {
    if ((rc = check_table(prefix_table, prefix_pages, prefix_pages, "prefix_table")) != DQG_OK) return rc;
    if (prefix_pages * pool.page_size < prefix_len)
      return api_fail(DQG_ERR_INVALID, "prefix_len=%lld positions exceed the prefix's %lld pages of %d",
                      (ll)prefix_len, (ll)prefix_pages, pool.page_size);
  }
  if ((rc = check_ptr(kv_lens, 4, "kv_lens")) != DQG_OK) return rc;
  if ((rc = check_ptr(out, 16, "out")) != DQG_OK) return rc;
  if ((rc = check_scale(scale)) != DQG_OK) return rc;
  if ((rc = check_workspace(workspace, workspace_bytes, need)) != DQG_OK) return rc;
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  dqg::DecodeArgs d;
  std::memset(&d, 0, sizeof(d));
  d.workspace = workspace;
  d.starved = starved;
  d.wait_ns = wait_ns;
  d.prefix_len = static_cast<int>(prefix_len);
  d.prefix_table = prefix_table;
  CUtensorMap qmap, kmap, vmap;
  if (prefix_len > 0 && !dqg::prefix_streamed(static_cast<int>(n_seqs), static_cast<int>(n_q_heads), pool.n_kv_heads,
                                              pool.D, static_cast<int>(prefix_len))) {
    dqg::PromptArgs a;
    std::memset(&a, 0, sizeof(a));
    a.table = prefix_table;
    a.table_stride = prefix_pages;
    a.table_width = static_cast<int>(prefix_pages);
    // The decode kernel's scratch first, the prefix's pieces behind it.
    a.workspace = static_cast<uint8_t*>(workspace) +
                  dqg::paged_decode_workspace(static_cast<int>(n_seqs), static_cast<int>(n_q_heads),
                                              pool.n_kv_heads, pool.D, static_cast<int>(prefix_len), sms);
    a.B = 1;
    a.T = static_cast<int>(n_seqs);
    a.hq = static_cast<int>(n_q_heads);
    a.scale_log2 = static_cast<float>(scale * kLog2e);
    a.prefix_len = static_cast<int>(prefix_len);
    if ((rc = query_map(q, pool, n_seqs, n_q_heads, q_stride_seq, q_stride_head, &qmap)) != DQG_OK) return rc;
    if ((rc = pool_maps(pool, dqg::prompt_box_rows(pool.page_size), &kmap, &vmap)) != DQG_OK) return rc;
    const cudaError_t e = dqg::launch_prompt(pool, qmap, kmap, vmap, a, sms, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return api_cuda_fail(e, "shared_prefix_attention launch");
    d.prefix = dqg::prefix_pieces(a, pool, sms);
  }
  if ((rc = pool_maps(pool, dqg::paged_decode_box_rows(pool.page_size), &kmap, &vmap)) != DQG_OK) return rc;
  d.q = q;
  d.q_stride_seq = q_stride_seq;
  d.q_stride_head = q_stride_head;
  d.table = block_table;
  d.table_stride = table_stride;
  d.table_width = static_cast<int>(table_width);
  d.lens = kv_lens;
  d.out = out;
  d.B = static_cast<int>(n_seqs);
  d.hq = static_cast<int>(n_q_heads);
  d.scale_log2 = static_cast<float>(scale * kLog2e);
  const cudaError_t e = dqg::launch_paged_decode(pool, kmap, vmap, d, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(e, "shared_prefix_attention launch");
  return api_ok();
}
}  // namespace

extern "C" {

int dqg_shared_prefix_attention(const void* q, int64_t q_stride_seq, int64_t q_stride_head, int64_t n_seqs,
                                int64_t n_q_heads, const dqg_paged_kv* kv, const int32_t* prefix_table,
                                int64_t prefix_pages, int64_t prefix_len, const int32_t* block_table,
                                int64_t table_width, int64_t table_stride, const int32_t* kv_lens,
                                float scale, void* out, void* workspace, uint64_t workspace_bytes,
                                void* stream) {
  return shared_prefix(q, q_stride_seq, q_stride_head, n_seqs, n_q_heads, kv, prefix_table, prefix_pages,
                       prefix_len, block_table, table_width, table_stride, kv_lens, scale, out, workspace,
                       workspace_bytes, 0, 0, stream);
}

int dqg_debug_paged_starved(const void* q, int64_t q_stride_seq, int64_t q_stride_head, int64_t n_seqs,
                            int64_t n_q_heads, const dqg_paged_kv* kv, const int32_t* prefix_table,
                            int64_t prefix_pages, int64_t prefix_len, const int32_t* block_table,
                            int64_t table_width, int64_t table_stride, const int32_t* kv_lens, float scale,
                            void* out, void* workspace, uint64_t workspace_bytes, uint32_t starved,
                            uint64_t wait_ns, void* stream) {
  if (wait_ns < 1000000ull || wait_ns > 1000000000ull)
    return api_fail(DQG_ERR_INVALID, "wait_ns must be in [1 ms, 1 s], got %llu", (unsigned long long)wait_ns);
  if (starved < 1 || starved > 31)
    return api_fail(DQG_ERR_INVALID, "starved must be in [1, 31], got %u", starved);
  return shared_prefix(q, q_stride_seq, q_stride_head, n_seqs, n_q_heads, kv, prefix_table, prefix_pages,
                       prefix_len, block_table, table_width, table_stride, kv_lens, scale, out, workspace,
                       workspace_bytes, starved, wait_ns, stream);
}

}  // extern "C"
