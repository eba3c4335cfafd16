// The draw of one token from each row of logits. No reference counterpart.
//
//   w_i = exp((l_i - max l) / T),  W_i = round(2^44 w_i)
//   kept: rank(i) < top_k, sum of W ranked before < top_p * sum over top_k, w_i >= min_p
//   token = first i, by index, with (sum of kept W up to i) > u * (their sum)
//
// Ranks are by logit, the lower index first. All sums are of 64-bit integers:
// exact, so that neither the order of summation nor the number of threads or
// CTAs changes a token.
//
// A cluster of up to eight CTAs takes a row; each holds a part of it in shared
// memory, and a thread a run of consecutive tokens of that. The logit at which
// top-k or top-p cuts is found digit by digit (11 bits of the ordered bits of
// its fp32 value; two digits say all of a 16-bit logit) from histograms of the
// tokens' number, or weight: a CTA's own first, whose bins in use are then added
// to a sum that every CTA has. So a digit costs one barrier of the cluster.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/dequant_b200.h"
#include "common.cuh"
#include "sampling.h"

namespace dqg {
namespace {

using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCtas = 8;
constexpr int kBins = 2048;
constexpr int kPer = kBins / kThreads;  // bins a thread
constexpr uint32_t kMinusInf = 0x007fffff;  // ordered bits of -inf

struct Params {
  SampleArgs a;
  int ctas;  // a row
  int run;   // tokens a thread: odd, so that reads of shared memory do not conflict
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Bits whose order is the values' (both zeros alike).
__device__ __forceinline__ uint32_t ordered(float v) {
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
    if (inf) return v == INFINITY ? 1.0 : 0.0;
    return v == -INFINITY ? 0.0 : exp((static_cast<double>(v) - m) * inv_t);
  }
  __device__ __forceinline__ u64 fixed(float v) const { return __double2ull_rn(weight(v) * 17592186044416.0); }
};

struct Shared {
  uint32_t own[3][kBins];     // this CTA's histogram: numbers, or 16 bits of the weights each
  uint32_t sum[2][3][kBins];  // the cluster's, in turn: numbers, or 24 bits of the weights each
  u64 scratch[kWarps];
  u64 total;                  // this CTA's part of a sum, read by its peers
  uint32_t largest, first, ties;
  uint32_t digit;             // of the cut
  u64 before, inside;         // ahead of its bin, and in it
};

__device__ __forceinline__ uint32_t peer_u32(const uint32_t* p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ u64 peer_u64(const u64* p, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(map_to_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void peer_add(uint32_t* p, int rank, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(map_to_rank(p, rank)), "r"(v) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  cluster_sync_all();
}

template <class F>
__device__ __forceinline__ uint32_t block_reduce(uint32_t v, u64* scratch, F f) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, off));
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = static_cast<uint32_t>(scratch[0]);
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v = f(v, static_cast<uint32_t>(scratch[w]));
  __syncthreads();
  return v;
}
// Sum of v over the threads before this one; *all: over the block.
__device__ __forceinline__ u64 block_scan(u64 v, u64* scratch, u64* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 sum = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += t;
  }
  if (lane == 31) scratch[warp] = sum;
  __syncthreads();
  u64 before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += scratch[w];
    total += scratch[w];
  }
  __syncthreads();
  *all = total;
  return before + sum - v;
}

struct Cut {  // kept: keys above, and the first `room` of those at it
  uint32_t key, room;
  bool all;  // room takes all of them
};

// One digit (bits above `shift`) of a cut: adds up the tokens' numbers or
// weights (add(i, digit)) in histograms, and returns in sh->digit, before and
// inside the bin that take(before the bin, in it) picks last, from the highest
// down. The buffers of sh->sum take turns; the next one is zeroed here.
template <class Add, class Take>
__device__ __forceinline__ void cut_digit(Shared* sh, int turn, int ctas, bool weighed, Add add, Take take) {
  const int arrays = weighed ? 3 : 1;
  for (int i = threadIdx.x; i < arrays * kBins; i += kThreads) (&sh->own[0][0])[i] = 0;
  for (int i = threadIdx.x; i < 3 * kBins; i += kThreads) (&sh->sum[turn ^ 1][0][0])[i] = 0;
  if (threadIdx.x == 0) sh->digit = 0;
  __syncthreads();
  add();
  __syncthreads();
  for (int bin = threadIdx.x; bin < kBins; bin += kThreads) {
    if (weighed) {
      const u64 w = sh->own[0][bin] + (static_cast<u64>(sh->own[1][bin]) << 16) + (static_cast<u64>(sh->own[2][bin]) << 32);
      if (w == 0) continue;
      for (int r = 0; r < ctas; ++r)
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const uint32_t part = static_cast<uint32_t>(w >> (24 * k)) & 0xffffffu;
          if (part) peer_add(&sh->sum[turn][k][bin], r, part);
        }
    } else if (sh->own[0][bin]) {
      for (int r = 0; r < ctas; ++r) peer_add(&sh->sum[turn][0][bin], r, sh->own[0][bin]);
    }
  }
  cluster_sync();
  // A thread's bins, the highest first.
  const int top = kBins - 1 - threadIdx.x * kPer;
  u64 in[kPer], mine = 0, all;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    in[k] = sh->sum[turn][0][top - k];
    if (weighed) in[k] += (static_cast<u64>(sh->sum[turn][1][top - k]) << 24) + (static_cast<u64>(sh->sum[turn][2][top - k]) << 48);
    mine += in[k];
  }
  u64 before = block_scan(mine, sh->scratch, &all);
  int best = -1;
  u64 best_before = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (in[k] && take(before)) {
      best = k;
      best_before = before;
    }
    before += in[k];
  }
  // The last bin taken has the highest rank from the top.
  const uint32_t rank = best < 0 ? 0 : threadIdx.x * kPer + best + 1;
  if (best >= 0) atomicMax(&sh->digit, rank);
  __syncthreads();
  const uint32_t last = sh->digit;
  __syncthreads();
  if (best >= 0 && rank == last) {
    sh->digit = kBins - last;
    sh->before = best_before;
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (k == best) sh->inside = in[k];
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ Params q) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const SampleArgs& p = q.a;
  Shared* sh = reinterpret_cast<Shared*>(smem_raw);
  float* x = reinterpret_cast<float*>(sh + 1);
  const int ctas = q.ctas, rank = static_cast<int>(cluster_ctarank()), row = blockIdx.x / ctas;
  const int lane = threadIdx.x & 31;
  const int slice = q.run * kThreads, base = rank * slice, n = max(0, min(slice, p.vocab - base));
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const float heat = p.temperatures ? __ldg(p.temperatures + row) : p.temperature;
  const int top_k = p.top_ks ? __ldg(p.top_ks + row) : p.top_k;
  const float top_p = p.top_ps ? __ldg(p.top_ps + row) : p.top_p;
  float min_p = p.min_ps ? __ldg(p.min_ps + row) : p.min_p;
  min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;

  // The row's part into shared memory; NaN becomes -inf.
  float largest = -INFINITY;
  {
    const T* from = static_cast<const T*>(p.logits) + row * p.row_stride + base;
    constexpr int kVec = 16 / sizeof(T);
    const int whole = reinterpret_cast<uintptr_t>(from) % 16 ? 0 : n / kVec * kVec;
    auto put = [&](int i, float v) {
      v = v == v ? v : -INFINITY;
      largest = fmaxf(largest, v);
      x[i] = v;
    };
    for (int i = threadIdx.x * kVec; i < whole; i += kThreads * kVec) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(from + i));
      const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int k = 0; k < kVec; ++k) put(i + k, to_float(v[k]));
    }
    for (int i = whole + threadIdx.x; i < n; i += kThreads) put(i, to_float(from[i]));
    for (int i = n + threadIdx.x; i < slice; i += kThreads) x[i] = -INFINITY;
  }
  for (int i = threadIdx.x; i < 3 * kBins; i += kThreads) (&sh->sum[0][0][0])[i] = 0;
  const auto most = [](uint32_t a, uint32_t b) { return max(a, b); };
  uint32_t top = block_reduce(ordered(largest), sh->scratch, most);
  if (threadIdx.x == 0) sh->largest = top;
  cluster_sync();
  for (int r = 0; r < ctas; ++r) top = max(top, peer_u32(&sh->largest, r));
  const float m = value_of(top);

  const int first = threadIdx.x * q.run;  // of this thread's tokens
  if (top <= kMinusInf) {
    if (rank == 0 && threadIdx.x == 0) {
      p.tokens[row] = -1;
      p.logprobs[row] = NAN;
    }
    cluster_sync();  // no CTA leaves while a peer reads from it
    return;
  }
  if (!(heat > 0.f)) {
    uint32_t at = 0xffffffffu;
    for (int j = q.run - 1; j >= 0; --j)
      if (x[first + j] == m) at = base + first + j;
    at = block_reduce(at, sh->scratch, [](uint32_t a, uint32_t b) { return min(a, b); });
    if (threadIdx.x == 0) sh->first = at;
    cluster_sync();
    if (rank == 0 && threadIdx.x == 0) {
      for (int r = 1; r < ctas; ++r) at = min(at, peer_u32(&sh->first, r));
      p.tokens[row] = at;
      p.logprobs[row] = 0.f;
    }
    cluster_sync();
    return;
  }
  const Row r{m, 1.0 / heat, m == INFINITY};
  constexpr int kDigits = sizeof(T) == 2 ? 2 : 3;
  // Bits of a 16-bit logit's key behind its second digit.
  auto filled = [](uint32_t key) { return kDigits == 2 && !(key >> 31) ? key | 0x3ffu : key; };
  auto shift_of = [](int digit) { return digit == 0 ? 21 : (digit == 1 ? 10 : 0); };

  Cut cut{0, 0, true};
  int turn = 0;
  if (top_k > 0 && top_k < p.vocab) {
    uint32_t want = top_k;
    for (int d = 0; d < kDigits; ++d, turn ^= 1) {
      const int shift = shift_of(d), mask = d == 2 ? 1023 : 2047;
      cut_digit(sh, turn, ctas, false, [&] {
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const uint32_t key = ordered(x[i]);
          if (d == 0 || (key ^ cut.key) >> shift_of(d - 1) == 0) atomicAdd(&sh->own[0][key >> shift & mask], 1u);
        }
      }, [&](u64 before) { return before < want; });
      cut.key |= sh->digit << shift;
      want -= static_cast<uint32_t>(sh->before);
      cut.all = want == sh->inside;
      __syncthreads();
    }
    cut.key = filled(cut.key);
    cut.room = want;
  }
  if (top_p < 1.f) {
    const Cut k = cut;
    const u64 w_k = k.key ? r.fixed(value_of(k.key)) : 0;
    // Of the tokens at top-k's cut those that it does not keep weigh nothing.
    const u64 left_out = k.key && !k.all ? (sh->inside - k.room) * w_k : 0;
    __syncthreads();  // the count at top-k's cut has been read
    uint32_t low = 0;
    u64 before = 0, inside = 0;
    double target = 0.0;
    for (int d = 0; d < kDigits; ++d, turn ^= 1) {
      const int shift = shift_of(d), mask = d == 2 ? 1023 : 2047;
      auto add = [&] {
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const float v = x[i];
          const uint32_t key = ordered(v);
          if (key < k.key || (d > 0 && (key ^ low) >> shift_of(d - 1))) continue;
          const u64 w = r.fixed(v);
          uint32_t* bin = &sh->own[0][key >> shift & mask];
          if (const uint32_t part = static_cast<uint32_t>(w) & 0xffffu) atomicAdd(bin, part);
          if (const uint32_t part = static_cast<uint32_t>(w >> 16) & 0xffffu) atomicAdd(bin + kBins, part);
          if (const uint32_t part = static_cast<uint32_t>(w >> 32)) atomicAdd(bin + 2 * kBins, part);
        }
      };
      if (d == 0) {
        // The first histogram's sum is top-k's: the target follows from it.
        cut_digit(sh, turn, ctas, true, add, [&](u64) { return true; });
        target = static_cast<double>(top_p) * static_cast<double>(sh->before + sh->inside - left_out);
        // The bin again, now that the target is known.
        const int at = kBins - 1 - threadIdx.x * kPer;
        u64 in[kPer], mine = 0, all;
#pragma unroll
        for (int b = 0; b < kPer; ++b) {
          in[b] = sh->sum[turn][0][at - b] + (static_cast<u64>(sh->sum[turn][1][at - b]) << 24) +
                  (static_cast<u64>(sh->sum[turn][2][at - b]) << 48);
          mine += in[b];
        }
        if (threadIdx.x == 0) sh->ties = 0;
        u64 ahead = block_scan(mine, sh->scratch, &all);
        u64 best_before = 0, best_in = 0;
        uint32_t best = 0;
#pragma unroll
        for (int b = 0; b < kPer; ++b) {
          if (in[b] && (ahead == 0 || static_cast<double>(ahead) < target)) {
            best = threadIdx.x * kPer + b + 1;
            best_before = ahead;
            best_in = in[b];
          }
          ahead += in[b];
        }
        if (best) atomicMax(&sh->ties, best);
        __syncthreads();
        if (best && best == sh->ties) {
          sh->digit = kBins - best;
          sh->before = best_before;
          sh->inside = best_in;
        }
        __syncthreads();
      } else {
        cut_digit(sh, turn, ctas, true, add, [&](u64 in_digit) {
          return before + in_digit == 0 || static_cast<double>(before + in_digit) < target;
        });
      }
      low |= sh->digit << shift;
      before += sh->before;
      inside = sh->inside;
      __syncthreads();
    }
    low = filled(low);
    // All tokens at this logit weigh the same: of them those that have less than
    // the target before them, and one at least where nothing is before.
    const u64 w = r.fixed(value_of(low));
    const u64 here = low == k.key && !k.all ? k.room : inside / w;
    const double most_of = (target - static_cast<double>(before)) / static_cast<double>(w);
    u64 few = most_of >= static_cast<double>(here) ? here : (most_of < 0.0 ? 0 : static_cast<u64>(most_of));
    while (few < here && static_cast<double>(before + few * w) < target) ++few;
    while (few > 0 && !(static_cast<double>(before + (few - 1) * w) < target)) --few;
    if (before == 0 && few == 0) few = 1;
    cut = Cut{low, static_cast<uint32_t>(few), few == inside / w};
  }

  // Tokens at the cut that this thread's come behind, where not all are kept.
  uint32_t ahead = 0;
  if (!cut.all) {
    uint32_t ties = 0;
    for (int j = 0; j < q.run; ++j) ties += ordered(x[first + j]) == cut.key;
    u64 all;
    ahead = static_cast<uint32_t>(block_scan(ties, sh->scratch, &all));
    if (threadIdx.x == 0) sh->ties = static_cast<uint32_t>(all);
    cluster_sync();
    for (int i = 0; i < rank; ++i) ahead += peer_u32(&sh->ties, i);
  }
  // W of a token if it is kept; *tie: tokens at the cut before it.
  auto kept = [&](float v, uint32_t* tie) -> u64 {
    const uint32_t key = ordered(v);
    const bool in = key > cut.key || (key == cut.key && (cut.all || *tie < cut.room));
    *tie += key == cut.key;
    if (!in || v == -INFINITY) return 0;
    const double w = r.weight(v);
    return w >= static_cast<double>(min_p) ? __double2ull_rn(w * 17592186044416.0) : 0;
  };
  u64 mine = 0, total = 0;
  {
    uint32_t tie = ahead;
    for (int j = 0; j < q.run; ++j) mine += kept(x[first + j], &tie);
  }
  u64 before = block_scan(mine, sh->scratch, &total);
  if (threadIdx.x == 0) sh->total = total;
  cluster_sync();
  total = 0;
  for (int i = 0; i < ctas; ++i) {
    const u64 t = peer_u64(&sh->total, i);
    if (i < rank) before += t;
    total += t;
  }
  // The first token whose running sum exceeds this integer (u total, held below total).
  const double u = fmaxf(__ldg(p.uniform + row), 0.f);
  u64 goal = static_cast<u64>(fmin(u * static_cast<double>(total), 9.0e18));
  if (goal >= total) goal = total - 1;
  const unsigned found = __ballot_sync(0xffffffffu, before <= goal && goal < before + mine);
  if (found) {
    // The warp looks through the one thread's tokens, 32 at a time.
    const int src = __ffs(found) - 1;
    before = __shfl_sync(0xffffffffu, before, src);
    uint32_t tie = __shfl_sync(0xffffffffu, ahead, src);
    const int from = __shfl_sync(0xffffffffu, first, src);
    for (int j0 = 0; j0 < q.run; j0 += 32) {
      const float v = j0 + lane < q.run ? x[from + j0 + lane] : -INFINITY;
      const unsigned at_cut = __ballot_sync(0xffffffffu, ordered(v) == cut.key);
      uint32_t mine_tie = tie + __popc(at_cut & ((1u << lane) - 1));
      const u64 w = kept(v, &mine_tie);
      tie += __popc(at_cut);
      u64 sum = w;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += t;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + sum > goal);
      if (past) {
        const int l = __ffs(past) - 1;
        if (lane == l) {
          p.tokens[row] = base + from + j0 + lane;
          p.logprobs[row] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(total)));
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  cluster_sync();
}

template <typename T>
cudaError_t launch(const SampleArgs& a, int num_sms, cudaStream_t stream) {
  Params p;
  p.a = a;
  // CTAs a row: enough for their shared memory to hold 16384 tokens each at
  // most, and, while they do not fill the GPU, until a CTA has 2048.
  int ctas = 1;
  while (ctas < kMaxCtas && (a.vocab > ctas * 16384 || (static_cast<int64_t>(a.rows) * ctas <= num_sms &&
                                                        a.vocab > ctas * 2048)))
    ctas *= 2;
  p.ctas = ctas;
  p.run = ((a.vocab + ctas - 1) / ctas + kThreads - 1) / kThreads | 1;
  const size_t smem = sizeof(Shared) + static_cast<size_t>(p.run) * kThreads * 4;
  static int configured[64] = {0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = 1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, p);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int num_sms, cudaStream_t stream) {
  if (a.type == DQG_FP32) return launch<float>(a, num_sms, stream);
  return a.type == DQG_BF16 ? launch<__nv_bfloat16>(a, num_sms, stream) : launch<__half>(a, num_sms, stream);
}

}  // namespace dqg
