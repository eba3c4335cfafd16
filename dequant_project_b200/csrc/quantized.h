// Host-side interface of the operators over a cache held in 8 bits
// (quantized_append.cu, expand_pages.cu, quantized_attention.cu), called by
// capi_quantized.cu.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "paged.h"

namespace dqg {

// Pools of codes [n_pages, n_kv_heads, page_size, D] (strides in bytes, D
// contiguous), of scales [n_pages, n_kv_heads, page_size / block] and of open
// blocks [n_open, n_kv_heads, block, D] (strides in elements).
struct QuantizedPool {
  void *k, *v;
  float *k_scale, *v_scale;
  void *k_open, *v_open;
  int64_t n_pages, page_stride, head_stride, row_stride;
  int64_t scale_page_stride, scale_head_stride;
  int64_t n_open, open_stride, open_head_stride;
  int n_kv_heads, page_size, D, block;
  bool e4m3, bf16;
};

// The sequences that a call reads or writes.
struct QuantizedSeqs {
  const int32_t* table;  // [B, table_stride]
  int64_t table_stride;
  int table_width;
  const int32_t* open_slots;  // [B]
  const int32_t* q_starts;    // [B + 1], or null
  const int32_t* lens;        // [B]
  int B;
};

struct QuantizedAppendArgs {
  const void* qkv;  // [T, (hq + 2 hkv) * D], rows qkv_stride apart
  int64_t qkv_stride;
  const float* cosv;  // [n_positions, rot / 2]
  const float* sinv;
  const int64_t* positions;  // [T]
  const void* q_norm;        // [D] or null
  const void* k_norm;
  void* q_out;  // [T, hq, D]
  int64_t n_positions;
  int T, hq, rot;
  float eps;
  bool interleaved;
};
cudaError_t launch_quantized_append(const QuantizedPool& pool, const QuantizedSeqs& seqs,
                                    const QuantizedAppendArgs& a, int num_sms, cudaStream_t stream);

cudaError_t launch_expand_pages(const QuantizedPool& pool, const QuantizedSeqs& seqs, int64_t n_pages,
                                void* k_out, void* v_out, int32_t* table_out, float* factors, int64_t scale_stride,
                                float scale_log2, cudaStream_t stream);

struct QuantizedAttentionArgs {
  const void* q;  // [B, hq, D], strides in elements
  int64_t q_stride_seq, q_stride_head;
  void* out;  // [B, hq, D] contiguous
  void* workspace;
  int hq;
  float scale;
  uint64_t wait_ns;  // limit of a wait; 0: the library's
  uint32_t starved;  // diagnostic: bit w < 7, consumer warp w gives up at once; bit 7, nothing is copied
};
constexpr int kQuantizedBoxRows = 16;  // of the tensor maps' boxes
size_t quantized_attention_workspace(int hq, int n_kv_heads, int D, int num_sms);
cudaError_t launch_quantized_attention(const QuantizedPool& pool, const QuantizedSeqs& seqs, const CUtensorMap& kmap,
                                       const CUtensorMap& vmap, const QuantizedAttentionArgs& a, int num_sms,
                                       cudaStream_t stream);

cudaError_t read_status_quantized_append(uint32_t* status, bool reset);
cudaError_t read_status_expand(uint32_t* status, bool reset);
cudaError_t read_status_quantized_attention(uint32_t* status, bool reset);

}  // namespace dqg
