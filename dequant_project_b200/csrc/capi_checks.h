// Argument checks and tensor maps that the entry points of the cache operators
// share (capi_paged.cu, capi_quantized.cu): each returns a status, with the
// message left for dqg_last_error.
#pragma once

#include <cmath>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/dequant_b200.h"
#include "paged.h"

namespace {

using dqg::api_cuda_fail;
using dqg::api_fail;
using dqg::api_ok;
using ll = long long;

inline int check_ptr(const void* p, size_t align, const char* name) {
  if (p == nullptr) return api_fail(DQG_ERR_INVALID, "%s must not be null", name);
  if (reinterpret_cast<uintptr_t>(p) % align)
    return api_fail(DQG_ERR_INVALID, "%s must be %d-byte aligned", name, static_cast<int>(align));
  return DQG_OK;
}

inline int check_heads(int64_t hq, int n_kv_heads) {
  if (hq < n_kv_heads || hq % n_kv_heads || hq / n_kv_heads > 128 || hq > 65535)
    return api_fail(DQG_ERR_INVALID,
                    "head counts (%lld query, %d KV) must give 1..128 query heads per KV head", (ll)hq,
                    n_kv_heads);
  return DQG_OK;
}

inline int check_scale(float scale) {
  if (!(scale > 0.f) || !std::isfinite(scale))
    return api_fail(DQG_ERR_INVALID, "scale must be positive and finite, got %g", scale);
  return DQG_OK;
}

// Rows and heads of the queries; dimensions of one element take any stride.
inline int check_query(const void* q, int64_t rows, int64_t heads, int64_t& stride0, int64_t& stride_head, int D) {
  const int rc = check_ptr(q, 16, "q");
  if (rc) return rc;
  if (heads == 1) stride_head = D;
  if (rows == 1) stride0 = heads * stride_head;
  if (stride_head < D || stride_head % 8 || stride0 < 1 || stride0 % 8 ||
      stride0 > (int64_t(1) << 38) || stride_head > (int64_t(1) << 31))
    return api_fail(DQG_ERR_INVALID, "q's strides must be multiples of 8 elements, got %lld and %lld",
                    (ll)stride0, (ll)stride_head);
  return DQG_OK;
}

inline int check_table(const int32_t* table, int64_t width, int64_t stride, const char* name) {
  const int rc = check_ptr(table, 4, name);
  if (rc) return rc;
  if (width < 1 || width > (int64_t(1) << 26) || stride < width)
    return api_fail(DQG_ERR_INVALID, "%s must hold at least one page a row (width %lld, stride %lld)", name,
                    (ll)width, (ll)stride);
  return DQG_OK;
}

inline int check_workspace(const void* ws, uint64_t have, uint64_t need) {
  if (need == 0) return DQG_OK;
  const int rc = check_ptr(ws, 16, "workspace");
  if (rc) return rc;
  if (have < need)
    return api_fail(DQG_ERR_INVALID, "workspace of %llu bytes needed, %llu given",
                    (unsigned long long)need, (unsigned long long)have);
  return DQG_OK;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);
// The driver's tensor-map encoder, looked up at run time.
inline EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return static_cast<EncodeFn>(nullptr);
    }
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

// A 4-dimensional map of `bytes`-byte values: sizes innermost first, strides in
// elements of the three outer dimensions, swizzled boxes of `values` values by
// `rows1` by `rows2` by `rows3`.
inline int make_map(CUtensorMap* map, const void* base, CUtensorMapDataType type, int bytes, const int64_t (&size)[4],
             const int64_t (&stride)[3], int values, int rows1, int rows2, int rows3,
                    CUtensorMapSwizzle swizzle, const char* name) {
  const EncodeFn fn = encode_fn();
  if (fn == nullptr) return api_fail(DQG_ERR_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
  cuuint64_t dims[4], strides[3];
  for (int i = 0; i < 4; ++i) dims[i] = static_cast<cuuint64_t>(size[i]);
  for (int i = 0; i < 3; ++i) strides[i] = static_cast<cuuint64_t>(stride[i]) * bytes;
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(values), static_cast<cuuint32_t>(rows1),
                             static_cast<cuuint32_t>(rows2), static_cast<cuuint32_t>(rows3)};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, type, 4, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return api_fail(DQG_ERR_INVALID, "%s: no tensor map for these sizes and strides (%d)", name,
                    static_cast<int>(r));
  return DQG_OK;
}

// A map of values of the pools' type, in boxes of 64 values a row.
inline int pool_map(CUtensorMap* map, const void* base, const dqg::PagedPool& pool, const int64_t (&size)[4],
             const int64_t (&stride)[3], int rows1, int rows2, int rows3, const char* name) {
  return make_map(map, base, pool.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, size,
                  stride, 64, rows1, rows2, rows3, CU_TENSOR_MAP_SWIZZLE_128B, name);
}

inline int pool_maps(const dqg::PagedPool& pool, int rows, CUtensorMap* k, CUtensorMap* v) {
  const int64_t size[4] = {pool.D, pool.page_size, pool.n_kv_heads, pool.n_pages};
  const int64_t stride[3] = {pool.row_stride, pool.head_stride, pool.page_stride};
  int rc = pool_map(k, pool.k, pool, size, stride, rows, 1, 1, "k_pages");
  if (rc) return rc;
  return pool_map(v, pool.v, pool, size, stride, rows, 1, 1, "v_pages");
}

// Queries [T, kv heads, g, D]: boxes of a tile's tokens, times the KV head's
// query heads, times 64 values.
inline int query_map(const void* q, const dqg::PagedPool& pool, int64_t T, int64_t hq, int64_t stride_row,
              int64_t stride_head, CUtensorMap* map) {
  const int64_t g = hq / pool.n_kv_heads;
  const int64_t size[4] = {pool.D, g, pool.n_kv_heads, T};
  const int64_t stride[3] = {stride_head, g * stride_head, stride_row};
  return pool_map(map, q, pool, size, stride, static_cast<int>(g), 1,
                  dqg::prompt_tokens_per_tile(static_cast<int>(hq), pool.n_kv_heads), "q");
}

constexpr double kLog2e = 1.4426950408889634;

inline int current(int* dev, int* sms) {
  const cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return api_cuda_fail(e, "cudaGetDevice");
  *sms = dqg::api_sm_count(*dev);
  if (*sms < 1) return api_fail(DQG_ERR_CUDA, "no SM count for device %d", *dev);
  return DQG_OK;
}

}  // namespace
