// Host-side interface of the paged-cache operators (paged_append.cu,
// prompt_attention.cu, paged_attention.cu), called by capi_paged.cu.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace dqg {

// A paged key/value cache: two pools of [n_pages, n_kv_heads, page_size, D]
// 16-bit values with the same strides (in elements, D contiguous).
struct PagedPool {
  const void* k;
  const void* v;
  int64_t n_pages, page_stride, head_stride, row_stride;
  int n_kv_heads, page_size, D;
  bool bf16;
};

struct AppendArgs {
  const void* qkv;              // [T, (hq + 2 hkv) * D], rows qkv_stride apart
  int64_t qkv_stride;
  const float* cosv;            // [n_positions, rot / 2]
  const float* sinv;
  const int64_t* positions;     // [T]
  const int64_t* slots;         // [T]: page * page_size + place in page; negative: not stored
  const void* q_norm;           // [D] or null
  const void* k_norm;
  void* q_out;                  // [T, hq, D]
  int64_t n_positions;
  int T, hq, rot;
  float eps;
  bool interleaved;
};
cudaError_t launch_paged_append(const PagedPool& pool, const AppendArgs& a, int num_sms,
                                cudaStream_t stream);

// Per-piece results of a prefix that a whole batch shares, in the prompt
// kernel's layout (prompt_attention.cu): merged into each sequence's own
// result by the decode kernels. S == 0: no prefix.
struct PrefixPieces {
  const float* o;     // [pair][kv head][S][D / 4][256] float4
  const float* ml;    // [pair][kv head][S][2][256]: reference of the weights (log2 units), sum
  int S, tq;          // pieces; sequences per 128-row tile
};

struct DecodeArgs {
  const void* q;                // [B, hq, D], strides in elements
  int64_t q_stride_seq, q_stride_head;
  const int32_t* table;         // [B, table_stride]
  int64_t table_stride;
  int table_width;              // pages a row of the table holds
  const int32_t* lens;          // [B]
  void* out;                    // [B, hq, D] contiguous
  void* workspace;
  int B, hq;
  float scale_log2;
  int prefix_len;               // a shared prefix: 0 for none
  const int32_t* prefix_table;
  PrefixPieces prefix;          // its pieces, where the prompt kernel took it
  uint64_t wait_ns;             // limit of a wait; 0: the library's
  uint32_t starved;             // diagnostic: bit w < 4, consumer warp w gives up at once; bit 4, nothing is copied
};
size_t paged_decode_workspace(int B, int hq, int n_kv_heads, int D, int prefix_len, int num_sms);
// Whether the decode kernel streams a prefix itself (else the prompt kernel
// takes it, and DecodeArgs::prefix its pieces).
bool prefix_streamed(int n_seqs, int hq, int n_kv_heads, int D, int prefix_len);
cudaError_t launch_paged_decode(const PagedPool& pool, const CUtensorMap& kmap,
                                const CUtensorMap& vmap, const DecodeArgs& a, int num_sms,
                                cudaStream_t stream);
// Rows of the tensor maps' boxes for the decode kernel's tiles.
int paged_decode_box_rows(int page_size);

struct PromptArgs {
  const int32_t* table;         // [B, table_stride] (the prefix: one row)
  int64_t table_stride;
  int table_width;
  const int32_t* q_starts;      // [B + 1]
  const int32_t* kv_lens;       // [B]
  void* out;                    // [T, hq, D] contiguous
  void* workspace;
  int B, T, hq;
  bool causal;
  float scale_log2;
  // A prefix: T rows see the same prefix_len keys of one table row; the
  // pieces go to the workspace as PrefixPieces describes. 0: a prompt.
  int prefix_len;
};
size_t prompt_workspace(int D, int num_sms);
size_t prefix_workspace(int n_seqs, int hq, int n_kv_heads, int D, int prefix_len, int num_sms);
int prefix_splits(int n_seqs, int hq, int n_kv_heads, int prefix_len, int num_sms);
int prompt_box_rows(int page_size);
int prompt_tokens_per_tile(int hq, int n_kv_heads);
// qmap: [T, kv heads, g, D] boxes of (tokens per tile, 1, g, 64).
cudaError_t launch_prompt(const PagedPool& pool, const CUtensorMap& qmap, const CUtensorMap& kmap,
                          const CUtensorMap& vmap, const PromptArgs& a, int num_sms,
                          cudaStream_t stream);
PrefixPieces prefix_pieces(const PromptArgs& a, const PagedPool& pool, int num_sms);

cudaError_t read_status_append(uint32_t* status, bool reset);
cudaError_t read_status_paged_decode(uint32_t* status, bool reset);
cudaError_t read_status_prompt(uint32_t* status, bool reset);

// Shared with capi.cu: the thread's error message and the SM count.
int api_fail(int code, const char* fmt, ...);
int api_ok();
int api_cuda_fail(cudaError_t e, const char* what);
int api_sm_count(int dev);

}  // namespace dqg
