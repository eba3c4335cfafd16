// The positions of some sequences of a cache held in 8 bits as 16-bit pages,
// one sequence's after the other's, with the table that says where they lie:
//
//   x = E(code * scale) in complete blocks, the open block's rows behind them,
//   zeros behind a sequence's end
//
// so that the operators over 16-bit pages can read them. Attention of prompts
// goes this way too, with keys as codes (exact in 16 bits) whose scales the
// prompt kernel applies to its scores: key values rounded to bf16 would move a
// score by 2^-9 of itself. In the product loop the codes would be expanded once
// for every 256 rows (and by warps that share their issue slots with the
// softmax that bounds it), here once for all.
//
// Bound by HBM: a byte read and two written a value. A block takes one page of
// one head, sixteen values a thread at a time.
#include <cstdint>

#include "paged_rope.cuh"
#include "quantized.cuh"

namespace dqg {
namespace {

constexpr int kThreads = 256;

struct Params {
  QuantizedPool pool;
  QuantizedSeqs seqs;
  void* k_out;
  void* v_out;
  int32_t* table_out;
  float* k_scales;       // keys as codes: their scales (see PromptArgs), or null
  int64_t scale_stride;
  int64_t n_pages;
  int page_shift, block_shift, len_limit;
};

__device__ __forceinline__ int pages_of(const Params& p, int b) {
  return (clamped_len(p.seqs.lens, b, p.len_limit) + (1 << p.page_shift) - 1) >> p.page_shift;
}

// Pages that there is no room for, and indexes out of range: one block looks
// at all sequences.
__device__ __forceinline__ void look_over(const Params& p, uint32_t* scratch) {
  int64_t before = 0;
  bool bad = false;
  for (int b0 = 0; b0 < p.seqs.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = b < p.seqs.B ? pages_of(p, b) : 0;
    int sum = c;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += t;
    }
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    int64_t at = before + sum - c;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) at += scratch[w];
      before += scratch[w];
    }
    __syncthreads();
    if (b >= p.seqs.B) continue;
    const int len = __ldg(p.seqs.lens + b);
    bad |= len < 0 || len > p.len_limit;
    for (int64_t i = at > p.n_pages ? 0 : p.n_pages - at; i < c; ++i) {
      p.table_out[static_cast<int64_t>(b) * p.seqs.table_width + i] = -1;
      bad = true;
    }
  }
  if (bad) atomicOr(&g_status, kStatusBadIndex);
}

template <typename E, class Code, int D>
__global__ void __launch_bounds__(kThreads) expand_pages_kernel(const __grid_constant__ Params p) {
  __shared__ uint32_t scratch[kThreads / 32 + 2];
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int hkv = p.pool.n_kv_heads;
  const int64_t u = blockIdx.x / hkv;
  const int kvh = static_cast<int>(blockIdx.x - u * hkv);
  if (u == p.n_pages) {
    if (kvh == 0) look_over(p, scratch);
    return;
  }
  int64_t in = 0;
  const int b = find_unit(p.seqs.B, u, [&](int i) { return pages_of(p, i); }, scratch, &in);
  if (b < 0) return;
  const int page_size = 1 << p.page_shift, block = 1 << p.block_shift;
  const int len = clamped_len(p.seqs.lens, b, p.len_limit), base = static_cast<int>(in) << p.page_shift;
  const int done = len & ~(block - 1);
  int page = __ldg(p.seqs.table + b * p.seqs.table_stride + in);
  int64_t slot = __ldg(p.seqs.open_slots + b);
  const bool bad_page = (page < 0 || page >= p.pool.n_pages) && base < done;
  const bool bad_slot = (slot < 0 || slot >= p.pool.n_open) && done < len && base + page_size > done;
  if (threadIdx.x == 0) {
    if (kvh == 0) p.table_out[static_cast<int64_t>(b) * p.seqs.table_width + in] = static_cast<int32_t>(u);
    if (bad_page || bad_slot) atomicOr(&g_status, kStatusBadIndex);
  }
  const int n8 = bad_page ? 0 : min(page_size, max(0, done - base));  // rows in 8 bits
  const int n16 = bad_slot ? n8 : min(page_size, len - base);         // and open ones behind them
  const bool raw = p.k_scales != nullptr;
  if (raw) {
    float* to = p.k_scales + kvh * p.scale_stride + scaled_keys_begin(static_cast<int>(u - in), page_size, b) + base / 16;
    for (int i = threadIdx.x; i < page_size / 16; i += kThreads)
      to[i] = 16 * i < n8 ? __ldg(p.pool.k_scale + page * p.pool.scale_page_stride + kvh * p.pool.scale_head_stride +
                                  (16 * i >> p.block_shift))
                          : 1.f;
  }
  for (int which = 0; which < 2; ++which) {
    const uint8_t* codes = static_cast<const uint8_t*>(which ? p.pool.v : p.pool.k) + page * p.pool.page_stride +
                           kvh * p.pool.head_stride;
    const float* scales = (which ? p.pool.v_scale : p.pool.k_scale) + page * p.pool.scale_page_stride +
                          kvh * p.pool.scale_head_stride;
    const E* open = static_cast<const E*>(which ? p.pool.v_open : p.pool.k_open) + slot * p.pool.open_stride +
                    kvh * p.pool.open_head_stride;
    E* out = static_cast<E*>(which ? p.v_out : p.k_out) + ((u * hkv + kvh) << p.page_shift) * D;
    for (int i = threadIdx.x; i < page_size * (D / 16); i += kThreads) {
      const int row = i / (D / 16), c = i % (D / 16);
      uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
      if (row < n8) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(codes + row * p.pool.row_stride + c * 16));
        const float scale = raw && !which ? 1.f : __ldg(scales + (row >> p.block_shift));
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
        float f[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) Code::unpack4(ww[e], f + 4 * e);
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] *= scale;
        lo = pack8<E>(f);
        hi = pack8<E>(f + 8);
      } else if (base + row >= done && row < n16) {
        const uint4* from = reinterpret_cast<const uint4*>(open + (base + row - done) * D + c * 16);
        lo = from[0];
        hi = from[1];
      }
      uint4* to = reinterpret_cast<uint4*>(out + row * D + c * 16);
      to[0] = lo;
      to[1] = hi;
    }
  }
}

template <typename E, class Code>
cudaError_t launch(const Params& p, cudaStream_t stream) {
  const int64_t blocks = (p.n_pages + 1) * p.pool.n_kv_heads;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return p.pool.D == 128 ? cudaLaunchKernelEx(&cfg, expand_pages_kernel<E, Code, 128>, p)
                         : cudaLaunchKernelEx(&cfg, expand_pages_kernel<E, Code, 64>, p);
}

}  // namespace

cudaError_t launch_expand_pages(const QuantizedPool& pool, const QuantizedSeqs& seqs, int64_t n_pages, void* k_out,
                                void* v_out, int32_t* table_out, float* k_scales, int64_t scale_stride,
                                cudaStream_t stream) {
  Params p;
  p.k_scales = k_scales;
  p.scale_stride = scale_stride;
  p.pool = pool;
  p.seqs = seqs;
  p.k_out = k_out;
  p.v_out = v_out;
  p.table_out = table_out;
  p.n_pages = n_pages;
  p.page_shift = p.block_shift = 0;
  while ((1 << p.page_shift) < pool.page_size) ++p.page_shift;
  while ((1 << p.block_shift) < pool.block) ++p.block_shift;
  const int64_t limit = static_cast<int64_t>(seqs.table_width) * pool.page_size;
  p.len_limit = limit < (1 << 30) ? static_cast<int>(limit) : 1 << 30;
  if (pool.bf16)
    return pool.e4m3 ? launch<__nv_bfloat16, E4m3>(p, stream) : launch<__nv_bfloat16, Int8>(p, stream);
  return pool.e4m3 ? launch<__half, E4m3>(p, stream) : launch<__half, Int8>(p, stream);
}

}  // namespace dqg

DQG_STATUS_READER(read_status_expand)
