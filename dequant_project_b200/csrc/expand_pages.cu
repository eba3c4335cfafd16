// The positions of some sequences of a cache held in 8 bits as 16-bit pages,
// one sequence's after the other's, with the table that says where they lie:
//
//   x = E(code * scale) in complete blocks, the open block's rows behind them,
//   zeros behind a sequence's end
//
// so that the operators over 16-bit pages can read them. Attention of prompts
// goes this way too, with keys as codes (exact in 16 bits) whose scales the
// prompt kernel applies to its scores: key values rounded to bf16 would move a
// score by 2^-9 of itself. Values become codes times the power of two at or below
// the scale, exact too but for small ones in fp16: powers below 2^-24 (int8) or
// 2^-15 (e4m3, whose least code is 2^-9) give numbers below its normal ones, off by
// up to 2^-25. What is left of the scale, in [1, 2), goes to the softmax's weights
// (rounded values cost as much precision as the weights' rounding does: fp16 error
// 3.2e-4 instead of 2.5e-4). In the product loop the codes would be expanded once
// for every 256 rows (and by warps that share their issue slots with the softmax
// that bounds it), here once for all.
//
// Bound by HBM: a byte read and two written a value. A block takes one page of
// as many heads as give its threads work (7000 positions of 8 heads in pages of 16
// 9.4 us instead of 12.0), sixteen keys and values a thread at a time. 2048
// positions of 32 heads of 128 (17 MB read, 34 written) take 11 us in a stream of
// calls, 4.5 TB/s, 30000 of 8 heads 35 us, 5.3 TB/s: the writes stay in L2 at
// first, the loads' latency bounds the short ones (7 cycles a warp's instruction).
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
  float* factors;        // keys and values as codes: what goes with them (see PromptArgs), or null
  float log_unit;        // what the logarithms of values' factors are multiplied by; 0: values whole
  int64_t scale_stride;
  int64_t n_pages;
  int page_shift, block_shift, len_limit, heads;
};

// The power of two at or below a scale (the scale itself where there is none).
__device__ __forceinline__ float power_of(float scale) {
  const uint32_t u = __float_as_uint(scale);
  return u >= 0x00800000u && u < 0x7f800000u ? __uint_as_float(u & 0x7f800000u) : scale;
}

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

// (Eight blocks an SM, so 32 registers, for which int8's four variants spill 12
// bytes. With six the expansion alone would be faster, 10.6 us instead of 11.2 for
// 2048 positions of 32 heads, but the prompt kernel behind it starts later: 78.3 us
// a call instead of 76.1.)
template <typename E, class Code, int D>
__global__ void __launch_bounds__(kThreads, 8) expand_pages_kernel(const __grid_constant__ Params p) {
  __shared__ uint32_t scratch[kThreads / 32 + 2];
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  // `heads` KV heads of a page a block, as many as give its threads work.
  const int hkv = p.pool.n_kv_heads, groups = (hkv + p.heads - 1) / p.heads;
  const int64_t u = blockIdx.x / groups;
  const int head0 = static_cast<int>(blockIdx.x - u * groups) * p.heads, heads = min(p.heads, hkv - head0);
  if (u == p.n_pages) {
    if (head0 == 0) look_over(p, scratch);
    return;
  }
  int64_t in = 0;
  const int b = find_unit(p.seqs.B, u, [&](int i) { return pages_of(p, i); }, scratch, &in);
  if (b < 0) return;
  const int page_size = 1 << p.page_shift, block = 1 << p.block_shift;
  const int len = clamped_len(p.seqs.lens, b, p.len_limit), base = static_cast<int>(in) << p.page_shift;
  const int done = len & ~(block - 1);
  const int page = __ldg(p.seqs.table + b * p.seqs.table_stride + in);
  const int64_t slot = __ldg(p.seqs.open_slots + b);
  const bool bad_page = (page < 0 || page >= p.pool.n_pages) && base < done;
  const bool bad_slot = (slot < 0 || slot >= p.pool.n_open) && done < len && base + page_size > done;
  if (threadIdx.x == 0 && head0 == 0) {
    p.table_out[static_cast<int64_t>(b) * p.seqs.table_width + in] = static_cast<int32_t>(u);
    if (bad_page || bad_slot) atomicOr(&g_status, kStatusBadIndex);
  }
  const int n8 = bad_page ? 0 : min(page_size, max(0, done - base));  // rows in 8 bits
  const int n16 = bad_slot ? n8 : min(page_size, len - base);         // and open ones behind them
  const bool raw = p.factors != nullptr;
  if (raw) {
    // (Behind the sequence's end up to a multiple of eight: read with the rest.)
    const int parts = base + page_size < len ? page_size / 16 : (base + page_size + 127) / 128 * 8 - base / 16;
    for (int n = threadIdx.x; n < parts * heads; n += kThreads) {
      const int kvh = head0 + n / parts, i = n % parts, s = base / 16 + i;
      const int64_t at = page * p.pool.scale_page_stride + kvh * p.pool.scale_head_stride + (16 * i >> p.block_shift);
      float f = 1.f;
      if (16 * i < n8 && p.log_unit > 0.f) {
        const float scale = __ldg(p.pool.v_scale + at), power = power_of(scale);
        if (power != scale && scale == scale) f = scale / power;  // (exact)
      }
      float* to = p.factors + 4 * (kvh * p.scale_stride + scaled_keys_begin(static_cast<int>(u - in), page_size, b)) +
                  s / 8 * 32 + s % 8;
      to[0] = 16 * i < n8 ? __ldg(p.pool.k_scale + at) : 1.f;
      to[8] = log2f(f) * p.log_unit;
      to[16] = 1.f / f;
    }
  }
  for (int n = threadIdx.x; n < heads << p.page_shift << (D == 128 ? 3 : 2); n += kThreads) {
    constexpr int kChunks = D / 16;
    const int row = (n / kChunks) & (page_size - 1), c = n % kChunks, kvh = head0 + (n / kChunks >> p.page_shift);
    uint4 got[2][2] = {};  // of keys and of values: codes, or 16 values
    float scale[2];
    const bool in8 = row < n8;
    if (in8) {
      const int64_t at = page * p.pool.page_stride + kvh * p.pool.head_stride + row * p.pool.row_stride + c * 16;
      const int64_t scale_at = page * p.pool.scale_page_stride + kvh * p.pool.scale_head_stride + (row >> p.block_shift);
      got[0][0] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.pool.k) + at));
      got[1][0] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.pool.v) + at));
      scale[0] = raw ? 1.f : __ldg(p.pool.k_scale + scale_at);
      scale[1] = __ldg(p.pool.v_scale + scale_at);
      if (raw && p.log_unit > 0.f) scale[1] = power_of(scale[1]);
    } else if (base + row >= done && row < n16) {
      const int64_t at = slot * p.pool.open_stride + kvh * p.pool.open_head_stride + (base + row - done) * D + c * 16;
      const uint4* k = reinterpret_cast<const uint4*>(static_cast<const E*>(p.pool.k_open) + at);
      const uint4* v = reinterpret_cast<const uint4*>(static_cast<const E*>(p.pool.v_open) + at);
      got[0][0] = k[0];
      got[0][1] = k[1];
      got[1][0] = v[0];
      got[1][1] = v[1];
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (in8) {
        const uint32_t w[4] = {got[which][0].x, got[which][0].y, got[which][0].z, got[which][0].w};
        float f[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) Code::unpack4(w[e], f + 4 * e);
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] *= scale[which];
        got[which][0] = pack8<E>(f);
        got[which][1] = pack8<E>(f + 8);
      }
      uint4* to = reinterpret_cast<uint4*>(static_cast<E*>(which ? p.v_out : p.k_out) +
                                           (((u * hkv + kvh) << p.page_shift) + row) * D + c * 16);
      to[0] = got[which][0];
      to[1] = got[which][1];
    }
  }
}

template <typename E, class Code>
cudaError_t launch(const Params& p, cudaStream_t stream) {
  const int64_t blocks = (p.n_pages + 1) * ((p.pool.n_kv_heads + p.heads - 1) / p.heads);
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
                                void* v_out, int32_t* table_out, float* factors, int64_t scale_stride,
                                float scale_log2, cudaStream_t stream) {
  Params p;
  p.log_unit = scale_log2 > 1e-30f ? 1.f / scale_log2 : 0.f;
  p.factors = factors;
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
  p.heads = kThreads / (pool.page_size * (pool.D / 16));
  p.heads = p.heads < 1 ? 1 : (p.heads < pool.n_kv_heads ? p.heads : pool.n_kv_heads);
  const int64_t limit = static_cast<int64_t>(seqs.table_width) * pool.page_size;
  p.len_limit = limit < (1 << 30) ? static_cast<int>(limit) : 1 << 30;
  if (pool.bf16)
    return pool.e4m3 ? launch<__nv_bfloat16, E4m3>(p, stream) : launch<__nv_bfloat16, Int8>(p, stream);
  return pool.e4m3 ? launch<__half, E4m3>(p, stream) : launch<__half, Int8>(p, stream);
}

}  // namespace dqg

DQG_STATUS_READER(read_status_expand)
