// The draw of one token from each row of logits.
//
//   w_i = exp((l_i - max l) / T),  W_i = round(2^44 w_i)
//   kept: rank(i) < top_k, sum of W ranked before < top_p * sum over top_k, w_i >= min_p
//   token = first i, by index, with (sum of kept W up to i) > u * (their sum)
//
// Ranks are by logit, the lower index first. All sums are of 64-bit integers:
// exact, so that neither the order of summation nor the number of threads
// changes a token.
//
// A block takes a row. The logit at which top-k or top-p cuts is found digit by
// digit (8 bits of the ordered bits of its fp32 value) from histograms of the
// tokens' number and weight; of the tokens that have this very logit the first
// few are kept.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/dequant_b200.h"
#include "common.cuh"
#include "sampling.h"

namespace dqg {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMinusInf = 0x007fffff;  // ordered bits of -inf

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Bits whose order is the values' (both zeros alike, NaN as -inf).
__device__ __forceinline__ uint32_t ordered(float v) {
  if (!(v == v)) return kMinusInf;
  const uint32_t u = __float_as_uint(v + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

struct Row {
  double m, inv_t;
  bool inf;  // the largest logit is +inf
  __device__ __forceinline__ double weight(float v) const {
    if (inf) return isinf(v) && v > 0.f ? 1.0 : 0.0;
    return v == -INFINITY || !(v == v) ? 0.0 : exp((static_cast<double>(v) - m) * inv_t);
  }
};
__device__ __forceinline__ unsigned long long fixed(double w) { return __double2ull_rn(w * 17592186044416.0); }

struct Shared {
  uint32_t count[256], limb[4][256];  // 12 bits of the weights each
  unsigned long long sums[kWarps];
  uint32_t ties[kWarps];
  uint32_t digit, kept;
  unsigned long long before;
};

template <typename T, class F>
__device__ __forceinline__ T block_reduce(T v, T* scratch, F f) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, off));
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
  for (int w = 1; w < kWarps; ++w) v = f(v, scratch[w]);
  __syncthreads();
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs p) {
  __shared__ Shared sh;
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = p.vocab;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const float heat = p.temperatures ? __ldg(p.temperatures + row) : p.temperature;
  const int top_k = p.top_ks ? __ldg(p.top_ks + row) : p.top_k;
  const float top_p = p.top_ps ? __ldg(p.top_ps + row) : p.top_p;
  float min_p = p.min_ps ? __ldg(p.min_ps + row) : p.min_p;
  min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;

  uint32_t largest = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) largest = max(largest, ordered(to_float(x[i])));
  largest = block_reduce(largest, sh.ties, [](uint32_t a, uint32_t b) { return max(a, b); });
  if (largest <= kMinusInf) {
    if (threadIdx.x == 0) {
      p.tokens[row] = -1;
      p.logprobs[row] = NAN;
    }
    return;
  }
  if (!(heat > 0.f)) {
    uint32_t first = n;
    for (int i = threadIdx.x; i < n; i += kThreads)
      if (ordered(to_float(x[i])) == largest) first = min(first, static_cast<uint32_t>(i));
    first = block_reduce(first, sh.ties, [](uint32_t a, uint32_t b) { return min(a, b); });
    if (threadIdx.x == 0) {
      p.tokens[row] = first;
      p.logprobs[row] = 0.f;
    }
    return;
  }
  const Row r{value_of(largest), 1.0 / heat, value_of(largest) == INFINITY};
  const auto add = [](unsigned long long a, unsigned long long b) { return a + b; };

  // Kept: keys above `cut`, and the first `room` of those at it.
  uint32_t cut = 0, room = 0xffffffffu;
  if (top_k > 0 && top_k < n) {
    uint32_t want = top_k;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += kThreads) sh.count[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t key = ordered(to_float(x[i]));
        if (shift == 24 || (key ^ cut) >> (shift + 8) == 0) atomicAdd(sh.count + (key >> shift & 255), 1u);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        uint32_t left = want;
        int d = 255;
        while (sh.count[d] < left) left -= sh.count[d--];
        sh.digit = d;
        sh.kept = left;
      }
      __syncthreads();
      cut |= sh.digit << shift;
      want = sh.kept;
      __syncthreads();
    }
    room = want;
  }
  if (top_p < 1.f) {
    unsigned long long sum = 0;
    uint32_t at_cut = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = to_float(x[i]);
      const uint32_t key = ordered(v);
      if (key > cut) sum += fixed(r.weight(v));
      at_cut += key == cut;
    }
    sum = block_reduce(sum, sh.sums, add);
    at_cut = block_reduce(at_cut, sh.ties, [](uint32_t a, uint32_t b) { return a + b; });
    const uint32_t k_cut = cut, k_room = min(room, at_cut);
    if (k_room) sum += k_room * fixed(r.weight(value_of(cut)));
    const double target = static_cast<double>(top_p) * static_cast<double>(sum);
    uint32_t low = 0;
    unsigned long long before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += kThreads)
        sh.count[i] = sh.limb[0][i] = sh.limb[1][i] = sh.limb[2][i] = sh.limb[3][i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const float v = to_float(x[i]);
        const uint32_t key = ordered(v);
        if (key < k_cut || (shift < 24 && (key ^ low) >> (shift + 8))) continue;
        const unsigned long long w = fixed(r.weight(v));
        const int d = key >> shift & 255;
        atomicAdd(sh.count + d, 1u);
        for (int k = 0; k < 4; ++k) atomicAdd(sh.limb[k] + d, static_cast<uint32_t>(w >> (12 * k)) & 0xfffu);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        // The lowest digit in use whose tokens have less than the target before them.
        unsigned long long a = before;
        sh.digit = 255;
        for (int d = 255; d >= 0; --d) {
          if (sh.count[d] == 0) continue;
          if (!(static_cast<double>(a) < target) && a > 0) break;
          sh.digit = d;
          sh.before = a;
          sh.kept = sh.count[d];
          for (int k = 0; k < 4; ++k) a += static_cast<unsigned long long>(sh.limb[k][d]) << (12 * k);
        }
      }
      __syncthreads();
      low |= sh.digit << shift;
      before = sh.before;
      at_cut = sh.kept;
      __syncthreads();
    }
    // Of the tokens at this logit those that have less than the target before them.
    const uint32_t c = low == k_cut ? k_room : at_cut;
    const unsigned long long w = fixed(r.weight(value_of(low)));
    uint32_t few = c;
    if (w > 0) {
      const double most = (target - static_cast<double>(before)) / static_cast<double>(w);
      few = most >= c ? c : (most < 0 ? 0 : static_cast<uint32_t>(most));
      while (few < c && static_cast<double>(before + few * w) < target) ++few;
      while (few > 0 && !(static_cast<double>(before + (few - 1) * w) < target)) --few;
    }
    if (before == 0 && few == 0) few = 1;  // the first token is always kept
    cut = low;
    room = few;
  }

  // Warps take one contiguous part of the row each.
  const int part = (n + kThreads - 1) / kThreads * 32, lo = min(n, warp * part), hi = min(n, lo + part);
  uint32_t ties = 0;
  for (int i = lo + lane; i < hi; i += 32) ties += ordered(to_float(x[i])) == cut;
  for (int off = 16; off >= 1; off >>= 1) ties += __shfl_xor_sync(0xffffffffu, ties, off);
  if (lane == 0) sh.ties[warp] = ties;
  __syncthreads();
  uint32_t rank = 0;
  for (int w = 0; w < warp; ++w) rank += sh.ties[w];
  auto kept = [&](int i, uint32_t* rank) -> unsigned long long {
    const float v = i < hi ? to_float(x[i]) : -INFINITY;
    const uint32_t key = ordered(v);
    const unsigned tie = __ballot_sync(0xffffffffu, i < hi && key == cut);
    const bool in = key > cut || (key == cut && *rank + __popc(tie & ((1u << lane) - 1)) < room);
    *rank += __popc(tie);
    const double w = in && i < hi ? r.weight(v) : 0.0;
    return w >= static_cast<double>(min_p) ? fixed(w) : 0;
  };
  unsigned long long mine = 0;
  uint32_t at = rank;
  for (int i = lo; i < hi; i += 32) mine += kept(i + lane, &at);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
  if (lane == 0) sh.sums[warp] = mine;
  __syncthreads();
  unsigned long long total = 0, before = 0;
  for (int w = 0; w < kWarps; ++w) {
    total += sh.sums[w];
    if (w < warp) before += sh.sums[w];
  }
  const double u = static_cast<double>(fmaxf(__ldg(p.uniform + row), 0.f)) * static_cast<double>(total);
  int last = 0;  // the last warp that holds a kept token
  for (int w = 0; w < kWarps; ++w)
    if (sh.sums[w]) last = w;
  const bool here = mine > 0 && !(static_cast<double>(before) > u) &&
                    (static_cast<double>(before + mine) > u || warp == last);
  if (!here) return;
  at = rank;
  int token = -1;
  unsigned long long its = 0;
  for (int i = lo; i < hi; i += 32) {
    const unsigned long long w = kept(i + lane, &at);
    unsigned long long sum = w;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned long long t = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += t;
    }
    const unsigned past = __ballot_sync(0xffffffffu, w > 0 && static_cast<double>(before + sum) > u);
    const unsigned any = __ballot_sync(0xffffffffu, w > 0);
    if (any) {
      const int l = past ? __ffs(past) - 1 : 31 - __clz(any);
      token = i + l;
      its = __shfl_sync(0xffffffffu, w, l);
    }
    if (past) break;
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) {
    p.tokens[row] = token;
    p.logprobs[row] = static_cast<float>(log(static_cast<double>(its) / static_cast<double>(total)));
  }
}

template <typename T>
cudaError_t launch(const SampleArgs& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int num_sms, cudaStream_t stream) {
  (void)num_sms;
  if (a.type == DQG_FP32) return launch<float>(a, stream);
  return a.type == DQG_BF16 ? launch<__nv_bfloat16>(a, stream) : launch<__half>(a, stream);
}

}  // namespace dqg
