// extern "C" entry points of the operators over a cache held in 8 bits (declared
// in include/dequant_b200.h): argument checks and launches. Nothing here allocates
// device memory, synchronises or throws.
#include <cstdint>
#include <cstring>
#include <cuda_runtime.h>

#include "capi_checks.h"
#include "quantized.h"

namespace {

int check_stride(int64_t stride, int64_t least, int64_t multiple, const char* name) {
  if (stride < least || stride % multiple || stride > (int64_t(1) << 38))
    return api_fail(DQG_ERR_INVALID, "%s must be a multiple of %lld and at least %lld, got %lld", name, (ll)multiple,
                    (ll)least, (ll)stride);
  return DQG_OK;
}

// The cache's description, checked; *pool is what the launchers take.
int check_quantized(const dqg_quantized_kv* kv, dqg::QuantizedPool* pool) {
  if (kv == nullptr) return api_fail(DQG_ERR_INVALID, "kv must not be null");
  const void* ptrs[6] = {kv->k, kv->v, kv->k_scale, kv->v_scale, kv->k_open, kv->v_open};
  const char* names[6] = {"k", "v", "k_scale", "v_scale", "k_open", "v_open"};
  const size_t align[6] = {16, 16, 4, 4, 16, 16};
  int rc = DQG_OK;
  for (int i = 0; i < 6; ++i)
    if ((rc = check_ptr(ptrs[i], align[i], names[i])) != DQG_OK) return rc;
  if (kv->codes != DQG_INT8 && kv->codes != DQG_E4M3)
    return api_fail(DQG_ERR_INVALID, "codes must be DQG_INT8 or DQG_E4M3, got %d", kv->codes);
  if (kv->dtype != DQG_FP16 && kv->dtype != DQG_BF16)
    return api_fail(DQG_ERR_INVALID, "dtype must be DQG_FP16 or DQG_BF16, got %d", kv->dtype);
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return api_fail(DQG_ERR_UNSUPPORTED, "paged operators handle head_dim 64 and 128, got %lld", (ll)kv->head_dim);
  const int64_t ps = kv->page_size;
  if (ps < 16 || ps > 256 || (ps & (ps - 1)))
    return api_fail(DQG_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256, got %lld", (ll)ps);
  if ((kv->block != 16 && kv->block != 32 && kv->block != 64) || kv->block > ps)
    return api_fail(DQG_ERR_UNSUPPORTED, "block must be 16, 32 or 64 and at most a page, got %lld", (ll)kv->block);
  if (kv->n_kv_heads < 1 || kv->n_kv_heads > 1024)
    return api_fail(DQG_ERR_INVALID, "n_kv_heads must be in [1, 1024], got %lld", (ll)kv->n_kv_heads);
  if (kv->n_pages < 1 || kv->n_pages > (int64_t(1) << 30))
    return api_fail(DQG_ERR_INVALID, "n_pages must be in [1, 2^30], got %lld", (ll)kv->n_pages);
  if (kv->n_open < 1 || kv->n_open > (int64_t(1) << 30))
    return api_fail(DQG_ERR_INVALID, "n_open must be in [1, 2^30], got %lld", (ll)kv->n_open);
  // A dimension of one element has no stride to speak of.
  const int64_t d = kv->head_dim, parts = ps / kv->block;
  const bool heads = kv->n_kv_heads > 1, pages = kv->n_pages > 1, opens = kv->n_open > 1;
  dqg::QuantizedPool p;
  p.row_stride = kv->row_stride;
  p.head_stride = heads ? kv->head_stride : kv->row_stride;
  p.page_stride = pages ? kv->page_stride : kv->row_stride;
  p.scale_head_stride = heads ? kv->scale_head_stride : parts;
  p.scale_page_stride = pages ? kv->scale_page_stride : parts;
  p.open_head_stride = heads ? kv->open_head_stride : kv->block * d;
  p.open_stride = opens ? kv->open_stride : kv->block * d;
  if ((rc = check_stride(p.row_stride, d, 16, "the codes' row stride")) != DQG_OK ||
      (rc = check_stride(p.head_stride, d, 16, "the codes' head stride")) != DQG_OK ||
      (rc = check_stride(p.page_stride, d, 16, "the codes' page stride")) != DQG_OK ||
      (rc = check_stride(p.scale_head_stride, parts, 1, "the scales' head stride")) != DQG_OK ||
      (rc = check_stride(p.scale_page_stride, parts, 1, "the scales' page stride")) != DQG_OK ||
      (rc = check_stride(p.open_head_stride, kv->block * d, 8, "the open blocks' head stride")) != DQG_OK ||
      (rc = check_stride(p.open_stride, kv->block * d, 8, "the open blocks' stride")) != DQG_OK)
    return rc;
  p.k = kv->k;
  p.v = kv->v;
  p.k_scale = kv->k_scale;
  p.v_scale = kv->v_scale;
  p.k_open = kv->k_open;
  p.v_open = kv->v_open;
  p.n_pages = kv->n_pages;
  p.n_open = kv->n_open;
  p.n_kv_heads = static_cast<int>(kv->n_kv_heads);
  p.page_size = static_cast<int>(ps);
  p.D = static_cast<int>(d);
  p.block = static_cast<int>(kv->block);
  p.e4m3 = kv->codes == DQG_E4M3;
  p.bf16 = kv->dtype == DQG_BF16;
  *pool = p;
  return DQG_OK;
}

int check_expanded(int64_t n_seqs, int64_t n_pages) {
  if (n_seqs < 0 || n_seqs > (1 << 20)) return api_fail(DQG_ERR_INVALID, "n_seqs=%lld out of range", (ll)n_seqs);
  if (n_pages < 0 || n_pages > (1 << 24)) return api_fail(DQG_ERR_INVALID, "n_pages=%lld out of range", (ll)n_pages);
  return DQG_OK;
}

int check_seqs(const int32_t* table, int64_t width, int64_t stride, const int32_t* open_slots, const int32_t* lens,
               int64_t n_seqs, dqg::QuantizedSeqs* seqs) {
  int rc = check_table(table, width, stride, "block_table");
  if (rc) return rc;
  if ((rc = check_ptr(open_slots, 4, "open_slots")) != DQG_OK) return rc;
  if ((rc = check_ptr(lens, 4, "kv_lens")) != DQG_OK) return rc;
  seqs->table = table;
  seqs->table_stride = stride;
  seqs->table_width = static_cast<int>(width);
  seqs->open_slots = open_slots;
  seqs->q_starts = nullptr;
  seqs->lens = lens;
  seqs->B = static_cast<int>(n_seqs);
  return DQG_OK;
}

}  // namespace

extern "C" {

int dqg_rope_quantized_append(const void* qkv, int64_t T, int64_t qkv_stride, int64_t n_q_heads,
                              const float* cos_table, const float* sin_table, int64_t n_positions,
                              int64_t rotary_dim, int interleaved, const int64_t* positions, const void* q_norm,
                              const void* k_norm, float eps, const dqg_quantized_kv* kv, const int32_t* block_table,
                              int64_t table_width, int64_t table_stride, const int32_t* open_slots,
                              const int32_t* q_starts, const int32_t* kv_lens, int64_t n_seqs, void* q_out,
                              void* stream) {
  dqg::QuantizedPool pool;
  dqg::QuantizedSeqs seqs;
  int rc = check_quantized(kv, &pool);
  if (rc) return rc;
  if ((rc = check_heads(n_q_heads, pool.n_kv_heads)) != DQG_OK) return rc;
  if (T < 0 || T > (1 << 28)) return api_fail(DQG_ERR_INVALID, "T=%lld out of range", (ll)T);
  if (n_seqs < 0 || n_seqs > (1 << 20)) return api_fail(DQG_ERR_INVALID, "n_seqs=%lld out of range", (ll)n_seqs);
  if (T == 0) return api_ok();
  const int64_t width = (n_q_heads + 2 * pool.n_kv_heads) * pool.D;
  if (qkv_stride < width || qkv_stride % 8)
    return api_fail(DQG_ERR_INVALID, "qkv's row stride must be a multiple of 8 and at least %lld, got %lld", (ll)width,
                    (ll)qkv_stride);
  if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > pool.D)
    return api_fail(DQG_ERR_INVALID, "rotary_dim must be even and in [2, head_dim], got %lld", (ll)rotary_dim);
  if (n_positions < 1) return api_fail(DQG_ERR_INVALID, "the cos/sin tables must hold at least one position");
  if ((q_norm == nullptr) != (k_norm == nullptr))
    return api_fail(DQG_ERR_INVALID, "q_norm and k_norm are given together or not at all");
  if (!(eps >= 0.f)) return api_fail(DQG_ERR_INVALID, "eps must be non-negative");
  const void* ptrs[7] = {qkv, cos_table, sin_table, positions, q_out, q_norm, k_norm};
  const char* names[7] = {"qkv", "cos", "sin", "positions", "q_out", "q_norm", "k_norm"};
  const size_t align[7] = {16, 4, 4, 8, 16, 16, 16};
  for (int i = 0; i < (q_norm ? 7 : 5); ++i)
    if ((rc = check_ptr(ptrs[i], align[i], names[i])) != DQG_OK) return rc;
  seqs = {};
  if (n_seqs > 0) {
    if ((rc = check_seqs(block_table, table_width, table_stride, open_slots, kv_lens, n_seqs, &seqs)) != DQG_OK)
      return rc;
    if ((rc = check_ptr(q_starts, 4, "q_starts")) != DQG_OK) return rc;
    seqs.q_starts = q_starts;
  }
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  dqg::QuantizedAppendArgs a;
  a.qkv = qkv;
  a.qkv_stride = qkv_stride;
  a.cosv = cos_table;
  a.sinv = sin_table;
  a.positions = positions;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.q_out = q_out;
  a.n_positions = n_positions;
  a.T = static_cast<int>(T);
  a.hq = static_cast<int>(n_q_heads);
  a.rot = static_cast<int>(rotary_dim);
  a.eps = eps;
  a.interleaved = interleaved != 0;
  const cudaError_t e = dqg::launch_quantized_append(pool, seqs, a, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(e, "rope_quantized_append launch");
  return api_ok();
}

int dqg_expand_pages(const dqg_quantized_kv* kv, const int32_t* block_table, int64_t table_width,
                     int64_t table_stride, const int32_t* open_slots, const int32_t* kv_lens, int64_t n_seqs,
                     int64_t n_pages, void* k_out, void* v_out, int32_t* table_out, void* stream) {
  dqg::QuantizedPool pool;
  dqg::QuantizedSeqs seqs;
  int rc = check_quantized(kv, &pool);
  if (rc) return rc;
  if ((rc = check_expanded(n_seqs, n_pages)) != DQG_OK) return rc;
  if (n_seqs == 0) return api_ok();
  if ((rc = check_seqs(block_table, table_width, table_stride, open_slots, kv_lens, n_seqs, &seqs)) != DQG_OK)
    return rc;
  if ((rc = check_ptr(table_out, 4, "table_out")) != DQG_OK) return rc;
  if (n_pages > 0 && ((rc = check_ptr(k_out, 16, "k_out")) != DQG_OK || (rc = check_ptr(v_out, 16, "v_out")) != DQG_OK))
    return rc;
  const cudaError_t e =
      dqg::launch_expand_pages(pool, seqs, n_pages, k_out, v_out, table_out, nullptr, 0, 0.f,
                               static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(e, "expand_pages launch");
  return api_ok();
}

}  // extern "C"

namespace {
// What a prompt call leaves between its kernels.
struct PromptScratch {
  uint64_t k, v, table, factors, pieces, bytes;  // offsets, and all of it
  int64_t scale_stride, n_pages;
};
PromptScratch prompt_scratch(const dqg::QuantizedPool& pool, int64_t n_seqs, int64_t table_width, int64_t n_pages,
                             int sms) {
  if (n_pages == 0) n_pages = 1;  // no position at all: a page for the maps, which nothing reads
  const auto up = [](uint64_t n) { return (n + 255) / 256 * 256; };
  const uint64_t pages = up(static_cast<uint64_t>(n_pages) * pool.n_kv_heads * pool.page_size * pool.D * 2);
  PromptScratch s;
  s.n_pages = n_pages;
  s.scale_stride = (n_pages * (pool.page_size / 16) + 7) / 8 * 8 + 8 * (n_seqs + 1);
  s.k = 0;
  s.v = pages;
  s.table = 2 * pages;
  s.factors = s.table + up(static_cast<uint64_t>(n_seqs) * table_width * 4);
  s.pieces = s.factors + up(static_cast<uint64_t>(s.scale_stride) * pool.n_kv_heads * 16);
  s.bytes = s.pieces + dqg::prompt_workspace(pool.D, sms);
  return s;
}
}  // namespace

extern "C" {

int dqg_quantized_prompt_workspace(const dqg_quantized_kv* kv, int64_t n_seqs, int64_t table_width, int64_t n_pages,
                                   uint64_t* bytes) {
  if (bytes == nullptr) return api_fail(DQG_ERR_INVALID, "bytes must not be null");
  dqg::QuantizedPool pool;
  int rc = check_quantized(kv, &pool);
  if (rc) return rc;
  if ((rc = check_expanded(n_seqs, n_pages)) != DQG_OK) return rc;
  if (table_width < 1 || table_width > (int64_t(1) << 26))
    return api_fail(DQG_ERR_INVALID, "table_width=%lld out of range", (ll)table_width);
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  *bytes = prompt_scratch(pool, n_seqs, table_width, n_pages, sms).bytes;
  return api_ok();
}

int dqg_quantized_prompt_attention(const void* q, int64_t q_stride_row, int64_t q_stride_head, int64_t T,
                                   int64_t n_q_heads, const dqg_quantized_kv* kv, const int32_t* block_table,
                                   int64_t table_width, int64_t table_stride, const int32_t* open_slots,
                                   const int32_t* q_starts, const int32_t* kv_lens, int64_t n_seqs, int64_t n_pages,
                                   int causal, float scale, void* out, void* workspace, uint64_t workspace_bytes,
                                   void* stream) {
  dqg::QuantizedPool pool;
  dqg::QuantizedSeqs seqs;
  int rc = check_quantized(kv, &pool);
  if (rc) return rc;
  if ((rc = check_heads(n_q_heads, pool.n_kv_heads)) != DQG_OK) return rc;
  if (T < 0 || T > (1 << 28)) return api_fail(DQG_ERR_INVALID, "T=%lld out of range", (ll)T);
  if ((rc = check_expanded(n_seqs, n_pages)) != DQG_OK) return rc;
  if (T == 0 || n_seqs == 0) return api_ok();
  if ((rc = check_query(q, T, n_q_heads, q_stride_row, q_stride_head, pool.D)) != DQG_OK) return rc;
  if ((rc = check_seqs(block_table, table_width, table_stride, open_slots, kv_lens, n_seqs, &seqs)) != DQG_OK)
    return rc;
  if ((rc = check_ptr(q_starts, 4, "q_starts")) != DQG_OK) return rc;
  if ((rc = check_ptr(out, 16, "out")) != DQG_OK) return rc;
  if ((rc = check_scale(scale)) != DQG_OK) return rc;
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  const PromptScratch s = prompt_scratch(pool, n_seqs, table_width, n_pages, sms);
  if ((rc = check_workspace(workspace, workspace_bytes, s.bytes)) != DQG_OK) return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int32_t* table = reinterpret_cast<int32_t*>(ws + s.table);
  dqg::PagedPool pages;
  pages.k = ws + s.k;
  pages.v = ws + s.v;
  pages.n_pages = s.n_pages;
  pages.row_stride = pool.D;
  pages.head_stride = static_cast<int64_t>(pool.page_size) * pool.D;
  pages.page_stride = pool.n_kv_heads * pages.head_stride;
  pages.n_kv_heads = pool.n_kv_heads;
  pages.page_size = pool.page_size;
  pages.D = pool.D;
  pages.bf16 = pool.bf16;
  CUtensorMap qmap, kmap, vmap;
  if ((rc = query_map(q, pages, T, n_q_heads, q_stride_row, q_stride_head, &qmap)) != DQG_OK) return rc;
  if ((rc = pool_maps(pages, dqg::prompt_box_rows(pages.page_size), &kmap, &vmap)) != DQG_OK) return rc;
  float* factors = reinterpret_cast<float*>(ws + s.factors);
  const float scale_log2 = static_cast<float>(scale * kLog2e);
  cudaError_t e = dqg::launch_expand_pages(pool, seqs, s.n_pages, ws + s.k, ws + s.v, table, factors, s.scale_stride,
                                           scale_log2, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(e, "quantized_prompt_attention launch");
  dqg::PromptArgs a;
  std::memset(&a, 0, sizeof(a));
  a.table = table;
  a.table_stride = table_width;
  a.table_width = static_cast<int>(table_width);
  a.q_starts = q_starts;
  a.kv_lens = kv_lens;
  a.out = out;
  a.workspace = ws + s.pieces;
  a.B = static_cast<int>(n_seqs);
  a.T = static_cast<int>(T);
  a.hq = static_cast<int>(n_q_heads);
  a.causal = causal != 0;
  a.scale_log2 = scale_log2;
  a.factors = factors;
  a.scale_stride = s.scale_stride;
  e = dqg::launch_prompt(pages, qmap, kmap, vmap, a, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(e, "quantized_prompt_attention launch");
  return api_ok();
}

int dqg_quantized_attention_workspace(int64_t n_seqs, int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
                                      uint64_t* bytes) {
  if (bytes == nullptr) return api_fail(DQG_ERR_INVALID, "bytes must not be null");
  if (head_dim != 64 && head_dim != 128)
    return api_fail(DQG_ERR_UNSUPPORTED, "paged operators handle head_dim 64 and 128, got %lld", (ll)head_dim);
  if (n_kv_heads < 1 || n_kv_heads > 1024)
    return api_fail(DQG_ERR_INVALID, "n_kv_heads must be in [1, 1024], got %lld", (ll)n_kv_heads);
  int rc = check_heads(n_q_heads, static_cast<int>(n_kv_heads));
  if (rc) return rc;
  if (n_seqs < 0 || n_seqs > (1 << 20)) return api_fail(DQG_ERR_INVALID, "n_seqs=%lld out of range", (ll)n_seqs);
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  *bytes = dqg::quantized_attention_workspace(static_cast<int>(n_q_heads), static_cast<int>(n_kv_heads),
                                              static_cast<int>(head_dim), sms);
  return api_ok();
}

}  // extern "C"

namespace {
int quantized_attention(const void* q, int64_t q_stride_seq, int64_t q_stride_head, int64_t n_seqs, int64_t n_q_heads,
                        const dqg_quantized_kv* kv, const int32_t* block_table, int64_t table_width,
                        int64_t table_stride, const int32_t* open_slots, const int32_t* kv_lens, float scale, void* out,
                        void* workspace, uint64_t workspace_bytes, uint32_t starved, uint64_t wait_ns, void* stream) {
  dqg::QuantizedPool pool;
  dqg::QuantizedSeqs seqs;
  int rc = check_quantized(kv, &pool);
  if (rc) return rc;
  if ((rc = check_heads(n_q_heads, pool.n_kv_heads)) != DQG_OK) return rc;
  if (n_seqs < 0 || n_seqs > (1 << 20)) return api_fail(DQG_ERR_INVALID, "n_seqs=%lld out of range", (ll)n_seqs);
  if (n_seqs == 0) return api_ok();
  if ((rc = check_query(q, n_seqs, n_q_heads, q_stride_seq, q_stride_head, pool.D)) != DQG_OK) return rc;
  if ((rc = check_seqs(block_table, table_width, table_stride, open_slots, kv_lens, n_seqs, &seqs)) != DQG_OK)
    return rc;
  if ((rc = check_ptr(out, 16, "out")) != DQG_OK) return rc;
  if ((rc = check_scale(scale)) != DQG_OK) return rc;
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  const uint64_t need = dqg::quantized_attention_workspace(static_cast<int>(n_q_heads), pool.n_kv_heads, pool.D, sms);
  if ((rc = check_workspace(workspace, workspace_bytes, need)) != DQG_OK) return rc;
  const int64_t size[4] = {pool.D, pool.page_size, pool.n_kv_heads, pool.n_pages};
  const int64_t stride[3] = {pool.row_stride, pool.head_stride, pool.page_stride};
  constexpr int rows = dqg::kQuantizedBoxRows;
  const CUtensorMapSwizzle swizzle = pool.D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  CUtensorMap kmap, vmap;
  if ((rc = make_map(&kmap, pool.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, size, stride, pool.D, rows, 1, 1, swizzle, "k")) !=
          DQG_OK ||
      (rc = make_map(&vmap, pool.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, size, stride, pool.D, rows, 1, 1, swizzle, "v")) !=
          DQG_OK)
    return rc;
  dqg::QuantizedAttentionArgs a;
  a.q = q;
  a.q_stride_seq = q_stride_seq;
  a.q_stride_head = q_stride_head;
  a.out = out;
  a.workspace = workspace;
  a.hq = static_cast<int>(n_q_heads);
  a.scale = scale;
  a.starved = starved;
  a.wait_ns = wait_ns;
  const cudaError_t e =
      dqg::launch_quantized_attention(pool, seqs, kmap, vmap, a, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(e, "quantized_attention launch");
  return api_ok();
}
}  // namespace

extern "C" {

int dqg_quantized_attention(const void* q, int64_t q_stride_seq, int64_t q_stride_head, int64_t n_seqs,
                            int64_t n_q_heads, const dqg_quantized_kv* kv, const int32_t* block_table,
                            int64_t table_width, int64_t table_stride, const int32_t* open_slots,
                            const int32_t* kv_lens, float scale, void* out, void* workspace, uint64_t workspace_bytes,
                            void* stream) {
  return quantized_attention(q, q_stride_seq, q_stride_head, n_seqs, n_q_heads, kv, block_table, table_width,
                             table_stride, open_slots, kv_lens, scale, out, workspace, workspace_bytes, 0, 0, stream);
}

int dqg_debug_quantized_starved(const void* q, int64_t q_stride_seq, int64_t q_stride_head, int64_t n_seqs,
                                int64_t n_q_heads, const dqg_quantized_kv* kv, const int32_t* block_table,
                                int64_t table_width, int64_t table_stride, const int32_t* open_slots,
                                const int32_t* kv_lens, float scale, void* out, void* workspace,
                                uint64_t workspace_bytes, uint32_t starved, uint64_t wait_ns, void* stream) {
  if (wait_ns < 1000000ull || wait_ns > 1000000000ull)
    return api_fail(DQG_ERR_INVALID, "wait_ns must be in [1 ms, 1 s], got %llu", (unsigned long long)wait_ns);
  if (starved < 1 || starved > 255) return api_fail(DQG_ERR_INVALID, "starved must be in [1, 255], got %u", starved);
  return quantized_attention(q, q_stride_seq, q_stride_head, n_seqs, n_q_heads, kv, block_table, table_width,
                             table_stride, open_slots, kv_lens, scale, out, workspace, workspace_bytes, starved,
                             wait_ns, stream);
}

}  // extern "C"
