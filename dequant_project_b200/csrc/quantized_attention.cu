// Decode attention over a cache held in 8 bits: one query token per sequence,
// lengths on the device, grouped KV heads.
//
//   o[b, h] = sum_t p_t s_v(t) code_v(t) / sum_t p_t,
//   p_t = exp(scale s_k(t) q[b, h] . code_k(t) - m)
//
// over the complete blocks of sequence b and then the 16-bit rows of its open
// block (s = 1); zero where there is none.
//
// A block takes one query head of one sequence, its warps every fourth
// position; a lane holds D / 32 values of the query and of the sum.
#include <cstdint>

#include "quantized.cuh"

namespace dqg {
namespace {

constexpr int kWarps = 4;

struct Params {
  QuantizedPool pool;
  QuantizedSeqs seqs;
  const void* q;
  void* out;
  int64_t q_stride_seq, q_stride_head;
  int hq, g, page_shift, block_shift, len_limit;
  float scale_log2;
};

template <typename E, class Code, int D>
__global__ void __launch_bounds__(32 * kWarps) quantized_attention_kernel(const __grid_constant__ Params p) {
  constexpr int kPer = D / 32;
  __shared__ float s_o[kWarps][D], s_m[kWarps], s_l[kWarps];
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int b = blockIdx.y, h = blockIdx.x, kvh = h / p.g, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = clamped_len(p.seqs.lens, b, p.len_limit), done = len >> p.block_shift << p.block_shift;
  if (threadIdx.x == 0 && __ldg(p.seqs.lens + b) != len) atomicOr(&g_status, kStatusBadIndex);
  const int64_t slot = __ldg(p.seqs.open_slots + b);
  const bool open = slot >= 0 && slot < p.pool.n_open;
  if (threadIdx.x == 0 && !open && done < len) atomicOr(&g_status, kStatusBadIndex);
  const E* q = static_cast<const E*>(p.q) + b * p.q_stride_seq + h * p.q_stride_head + lane * kPer;
  float qv[kPer], o[kPer], m = -INFINITY, l = 0.f;
  for (int i = 0; i < kPer; ++i) {
    qv[i] = Elem<E>::load(q + i) * p.scale_log2;
    o[i] = 0.f;
  }
  for (int t = warp; t < len; t += kWarps) {
    float k[kPer], v[kPer];
    if (t < done) {
      const int page = __ldg(p.seqs.table + b * p.seqs.table_stride + (t >> p.page_shift));
      const int row = t & ((1 << p.page_shift) - 1);
      const bool good = page >= 0 && page < p.pool.n_pages;
      if (!good && lane == 0) atomicOr(&g_status, kStatusBadIndex);
      const int64_t at = page * p.pool.page_stride + kvh * p.pool.head_stride + row * p.pool.row_stride + lane * kPer;
      const int64_t sc = page * p.pool.scale_page_stride + kvh * p.pool.scale_head_stride + (row >> p.block_shift);
      float f[4];
      for (int which = 0; which < 2; ++which) {
        const uint8_t* codes = static_cast<const uint8_t*>(which ? p.pool.v : p.pool.k);
        const float s = good ? __ldg((which ? p.pool.v_scale : p.pool.k_scale) + sc) : 0.f;
        uint32_t w = 0;
        if (good)
          for (int i = 0; i < kPer; ++i) w |= static_cast<uint32_t>(codes[at + i]) << (8 * i);
        Code::unpack4(w, f);
        for (int i = 0; i < kPer; ++i) (which ? v : k)[i] = f[i] * s;
      }
    } else {
      const int64_t at = slot * p.pool.open_stride + kvh * p.pool.open_head_stride + (t - done) * D + lane * kPer;
      for (int i = 0; i < kPer; ++i) {
        k[i] = open ? Elem<E>::load(static_cast<const E*>(p.pool.k_open) + at + i) : 0.f;
        v[i] = open ? Elem<E>::load(static_cast<const E*>(p.pool.v_open) + at + i) : 0.f;
      }
    }
    float s = 0.f;
    for (int i = 0; i < kPer; ++i) s = fmaf(qv[i], k[i], s);
    for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const float mx = fmaxf(m, s), f = exp2f(m - mx), w = exp2f(s - mx);
    l = fmaf(l, f, w);
    for (int i = 0; i < kPer; ++i) o[i] = fmaf(o[i], f, w * v[i]);
    m = mx;
  }
  for (int i = 0; i < kPer; ++i) s_o[warp][lane * kPer + i] = o[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += 32 * kWarps) {
    float mx = -INFINITY, den = 0.f, num = 0.f;
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_m[w]);
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_l[w] == 0.f ? 0.f : exp2f(s_m[w] - mx);
      den = fmaf(s_l[w], f, den);
      num = fmaf(s_o[w][i], f, num);
    }
    const float x = den == 0.f ? 0.f : num / den;
    static_cast<E*>(p.out)[(static_cast<int64_t>(b) * p.hq + h) * D + i] =
        reinterpret_cast<const E&>(static_cast<const uint16_t&>(static_cast<uint16_t>(Elem<E>::pack(x, 0.f))));
  }
}

template <typename E, class Code>
cudaError_t launch(const Params& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.hq, p.seqs.B);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return p.pool.D == 128 ? cudaLaunchKernelEx(&cfg, quantized_attention_kernel<E, Code, 128>, p)
                         : cudaLaunchKernelEx(&cfg, quantized_attention_kernel<E, Code, 64>, p);
}

}  // namespace

size_t quantized_attention_workspace(int, int, int, int, int) { return 16; }

cudaError_t launch_quantized_attention(const QuantizedPool& pool, const QuantizedSeqs& seqs,
                                       const QuantizedAttentionArgs& a, int num_sms, cudaStream_t stream) {
  (void)num_sms;
  Params p;
  p.pool = pool;
  p.seqs = seqs;
  p.q = a.q;
  p.out = a.out;
  p.q_stride_seq = a.q_stride_seq;
  p.q_stride_head = a.q_stride_head;
  p.hq = a.hq;
  p.g = a.hq / pool.n_kv_heads;
  p.page_shift = p.block_shift = 0;
  while ((1 << p.page_shift) < pool.page_size) ++p.page_shift;
  while ((1 << p.block_shift) < pool.block) ++p.block_shift;
  const int64_t limit = static_cast<int64_t>(seqs.table_width) * pool.page_size;
  p.len_limit = limit < (1 << 30) ? static_cast<int>(limit) : 1 << 30;
  p.scale_log2 = a.scale * 1.44269504f;
  if (pool.bf16)
    return pool.e4m3 ? launch<__nv_bfloat16, E4m3>(p, stream) : launch<__nv_bfloat16, Int8>(p, stream);
  return pool.e4m3 ? launch<__half, E4m3>(p, stream) : launch<__half, Int8>(p, stream);
}

}  // namespace dqg

DQG_STATUS_READER(read_status_quantized_attention)
