// The draw of one token from each row of logits. No reference counterpart.
//
//   w_i = exp((l_i - max l) / T),  W_i = round(2^44 w_i)
//   kept: rank(i) < top_k, sum of W ranked before < top_p * sum over top_k, w_i >= min_p
//   token = first i, by index, with (sum of kept W up to i) > u * (their sum)
//
// Ranks are by logit, the lower index first. All sums are of 64-bit integers:
// exact, so that neither the order of summation nor the number of threads or
// CTAs changes a token. A w is rounded once: by 2^-31 of itself, or by 2^-45 where
// that is more (half of a W's unit). The exponent is formed in pairs of fp32
// numbers, its fraction in 64ths from a table and the rest by a polynomial (a 64-bit
// exp took more than half of the time).
//
// A cluster of up to eight CTAs takes a row; each holds a part of it in shared
// memory, and a thread a run of consecutive tokens of that. The logit at which
// top-k or top-p cuts is found from histograms of the ordered bits of the
// logits (numbers, or weights), 1024 bins of equal width at a time, until a bin
// is one logit: a CTA's own histogram first, whose bins in use are then added to
// a sum that every CTA has, so that one barrier of the cluster is enough. What
// lies far below a cut stays out of the histograms: top-k's cut is above what
// the k-th largest of the threads' maxima is above, and top-p's above the
// largest of five weights that has top_p of the sum from it on. The tokens that
// are left, mostly a few, are listed once and read from there; up to 256 of them
// are not searched at all, but ranked by one CTA that compares each with all.
//
// Neither HBM nor arithmetic bounds it, but the chain of steps that each need
// the whole row's last (barriers are the largest stall: 5 cycles a warp's
// instruction): 64 rows of 128256 in fp16 with all parameters 29 to 37 us by
// the rows drawn (16.4 MB, 2.5 us), up to 50 where the cuts fall in flat places, one
// row of 32000 9 to 13 us, 256 rows of 32000 in fp32 33 us (without a cut: occupancy
// bounds that, two CTAs an SM and so two waves of them). Top-k alone (50) takes 17 us
// for the 64 rows; top-p of 0.9 over normal logits (deviation 3), whose cut lies among
// ten thousand tokens, 72 (114 with lists of 2048 a CTA, which do not hold them). A
// row a CTA with a 64-bit exp took 412 us, clusters 116, weights in pairs 61, short
// lists 42; rows kept in their own type, so that half the CTAs hold one and all 64
// rows run at once, 31.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "../../include/dequant_b200.h"
#include "common.cuh"
#include "sampling.h"

namespace dqg {
namespace {

using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCtas = 8;
constexpr int kBins = 1024;
constexpr int kPer = kBins / kThreads;  // bins a thread
constexpr int kListed = 6144;           // tokens that a CTA's list holds
constexpr int kDirect = 256;            // tokens of a row's lists that one CTA ranks
constexpr int kLevels = 5;              // weights 2^-4, 2^-7, 2^-10, 2^-13, 2^-16

struct Params {
  SampleArgs a;
  int ctas;  // a row
  int run;   // tokens a thread: an odd number of words, so that reads of shared memory do not conflict
};

// 2^(j / 64), as an integer of 44 fractional bits and as a float times 2^31.
struct Power {
  u64 fixed;
  float scaled, unused;
};
struct Powers {
  Power at[64];
};
constexpr Powers powers() {
  Powers t{};
  for (int j = 0; j < 64; ++j) {
    const double x = 0.693147180559945309417 * j / 64;
    double term = 1, sum = 1;
    for (int k = 1; k < 24; ++k) sum += term *= x / k;
    t.at[j] = Power{static_cast<u64>(sum * 17592186044416.0 + 0.5), static_cast<float>(sum * 2147483648.0), 0.f};
  }
  return t;
}
__device__ const Powers kPowers = powers();

// Types of logits, as a row is kept in shared memory: words of one or two.
template <typename T>
struct Logit;
template <>
struct Logit<float> {
  static constexpr int kDrop = 0;  // low bits of an fp32 value that these never use
  static constexpr uint32_t kLowest = 0xff800000u;
  static __device__ __forceinline__ float load(float v) { return v; }
  static __device__ __forceinline__ float store(float v) { return v; }
  // The larger of two words' values; NaN loses.
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float2 both(uint32_t w) { return make_float2(__uint_as_float(w), -INFINITY); }
};
template <>
struct Logit<__half> {
  static constexpr int kDrop = 13;
  static constexpr uint32_t kLowest = 0xfc00fc00u;
  static __device__ __forceinline__ float load(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half store(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(reinterpret_cast<const __half2&>(a), reinterpret_cast<const __half2&>(b));
    return reinterpret_cast<const uint32_t&>(m);
  }
  static __device__ __forceinline__ float2 both(uint32_t w) {
    return __half22float2(reinterpret_cast<const __half2&>(w));
  }
};
template <>
struct Logit<__nv_bfloat16> {
  static constexpr int kDrop = 16;
  static constexpr uint32_t kLowest = 0xff80ff80u;
  static __device__ __forceinline__ float load(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 store(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m =
        __hmax2(reinterpret_cast<const __nv_bfloat162&>(a), reinterpret_cast<const __nv_bfloat162&>(b));
    return reinterpret_cast<const uint32_t&>(m);
  }
  static __device__ __forceinline__ float2 both(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};

// f(logit, place) for the words from, from + step, ... of the first `count`
// tokens at x; kEven: count fills its words.
template <typename T, bool kEven, class F>
__device__ __forceinline__ void each_word(const T* x, int from, int step, int count, F f) {
  constexpr int kPack = 4 / sizeof(T);
#pragma unroll 4
  for (int i = from * kPack; i < count; i += step * kPack) {
    const float2 v = Logit<T>::both(*reinterpret_cast<const uint32_t*>(x + i));
    f(v.x, i);
    if (kPack == 2 && (kEven || i + 1 < count)) f(v.y, i + 1);
  }
}

// Integers whose order is the values' (both zeros alike), and back.
template <int kDrop>
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u >> 31 ? ~u : u | 0x80000000u) >> kDrop;
}
template <int kDrop>
__device__ __forceinline__ float value_of(uint32_t key) {
  const uint32_t u = key << kDrop;
  return __uint_as_float(u >> 31 ? u & 0x7fffffffu : ~(u | ((1u << kDrop) - 1)));
}

struct alignas(16) Shared {
  Power powers[64];
  uint32_t own[3][kBins];     // this CTA's histogram: numbers, or 16 bits of the weights each
  // The cluster's, of the bins that this CTA holds (every ctas-th; a CTA alone
  // has its own histogram), in turn: numbers, or 24 bits of the weights each.
  uint32_t sum[3][3][kBins / 2];
  uint16_t list[kListed];     // places in the CTA's part of the row
  u64 scratch[kWarps];
  u64 wide[kLevels + 2][kWarps];
  u64 parts[kLevels + 2];     // of sums and of a number of ties, read by the peers
  float largest;
  uint32_t first, cut_ties, listed;
  int limit;                  // place of the last token at the cut that is kept
  u64 total;
  uint32_t bin;               // of the cut
  u64 before, inside;         // ahead of it, and in it
};

struct Ranked {  // a token of a row's lists
  u64 w;
  float v;
  uint32_t place;
};
struct Ranks {  // of half of a row's tokens: those ahead of one
  u64 w;
  uint32_t greater, ties;
};

struct Weights {
  float m, high, low;  // the largest logit; log2(e) / T in two parts
  const Power* powers;
  // W of a logit (m finite). No branches: several tokens' chains run together.
  __device__ __forceinline__ u64 operator()(float v) const {
    // s + err = v - m and p + e = (v - m) log2(e) / T, in twice the precision.
    const float s = v - m, back = s - v;
    const float p = fmaxf(s * high, -48.f);
    const float err = (v - (s - back)) + (-m - back);
    const float e = fmaf(err, high, fmaf(s, low, fmaf(s, high, -p)));
    const float t = fmaf(p, 64.f, 12582912.f);  // 1.5 * 2^23: the fraction's last bit is one
    const int n = __float_as_int(t) - 0x4b400000;
    const float r = fmaf(t - 12582912.f, -1.f / 64.f, p) + e;  // 64ths out; at most 1/128
    // 2^r - 1
    const float q = r * fmaf(r, fmaf(r, fmaf(r, 9.6181291e-3f, 5.5504109e-2f), 2.4022651e-1f), 6.9314718e-1f);
    const Power w = powers[n & 63];
    const u64 one = w.fixed + (static_cast<long long>(__float2int_rn(q * w.scaled)) << 13);
    return p >= -46.f ? (((one << 1) >> -(n >> 6)) + 1) >> 1 : 0;
  }
};

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  cluster_sync_all();
}
template <typename V>
__device__ __forceinline__ V peer(const V* p, int rank) {
  V v;
  if constexpr (sizeof(V) == 8)
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(map_to_rank(p, rank)) : "memory");
  else
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(reinterpret_cast<uint32_t&>(v)) : "r"(map_to_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void peer_add(uint32_t* p, int rank, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(map_to_rank(p, rank)), "r"(v) : "memory");
}

template <typename V, class F>
__device__ __forceinline__ V block_reduce(V v, u64* scratch, F f) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, off));
  V* s = reinterpret_cast<V*>(scratch);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v = f(v, s[w]);
  __syncthreads();
  return v;
}
// f over what the cluster's CTAs have at p, and of the CTAs before `rank` alone
// (*before), `none` standing for no value. A lane a CTA.
template <typename V, class F>
__device__ __forceinline__ V cluster_reduce(const V* p, int ctas, V none, F f, int rank = 0, V* before = nullptr) {
  static_assert(kMaxCtas == 8, "eight lanes");
  const int r = threadIdx.x & 7;
  V v = r < ctas ? peer(p, r) : none, b = r < rank ? v : none;
#pragma unroll
  for (int off = 4; off >= 1; off >>= 1) {
    v = f(v, __shfl_xor_sync(0xffffffffu, v, off));
    if (before) b = f(b, __shfl_xor_sync(0xffffffffu, b, off));
  }
  if (before) *before = b;
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

// One round of a cut's search: histograms over bins that add() fills (tokens'
// numbers, or their weights), added up over the cluster; the bin that
// take(sum before it) takes last, from the highest down, goes to sh->bin, with
// sh->before and sh->inside. Three buffers of the cluster's sums take turns:
// a round's is read by the peers until they come to the next one's barrier, and
// zeroed in the round after that, before the barrier behind which it is used.
template <bool kWeighed, class Add, class Take>
__device__ __forceinline__ void search_round(Shared* sh, int round, int ctas, Add add, Take take) {
  constexpr int kArrays = kWeighed ? 3 : 1;
  auto& sum = sh->sum[round % 3];
  for (int i = threadIdx.x; i < kArrays * kBins; i += kThreads) (&sh->own[0][0])[i] = 0;
  if (threadIdx.x == 0) sh->bin = 0;
  __syncthreads();
  add();
  __syncthreads();
  u64 in[kPer], mine = 0, all;
  // A thread's bins, the highest first.
  const int top = kBins - 1 - threadIdx.x * kPer;
  if (ctas == 1) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      in[k] = sh->own[0][top - k];
      if (kWeighed) in[k] += (static_cast<u64>(sh->own[1][top - k]) << 16) + (static_cast<u64>(sh->own[2][top - k]) << 32);
    }
  } else {
    const int share = __ffs(ctas) - 1;
    for (int i = threadIdx.x; i < 3 * (kBins >> share); i += kThreads)
      sh->sum[(round + 1) % 3][i / (kBins >> share)][i % (kBins >> share)] = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int bin = threadIdx.x + k * kThreads, owner = bin & (ctas - 1), at = bin >> share;
      if (kWeighed) {
        const u64 w = sh->own[0][bin] + (static_cast<u64>(sh->own[1][bin]) << 16) + (static_cast<u64>(sh->own[2][bin]) << 32);
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          const uint32_t part = static_cast<uint32_t>(w >> (24 * j)) & 0xffffffu;
          if (part) peer_add(&sum[j][at], owner, part);
        }
      } else if (sh->own[0][bin]) {
        peer_add(&sum[0][at], owner, sh->own[0][bin]);
      }
    }
    cluster_sync();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int owner = (top - k) & (ctas - 1), at = (top - k) >> share;
      in[k] = peer(&sum[0][at], owner);
      if (kWeighed)
        in[k] += (static_cast<u64>(peer(&sum[1][at], owner)) << 24) + (static_cast<u64>(peer(&sum[2][at], owner)) << 48);
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) mine += in[k];
  u64 before = block_scan(mine, sh->scratch, &all);
  uint32_t best = 0;  // places from the top, and one
  u64 best_before = 0, best_in = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (in[k] && take(before)) {
      best = threadIdx.x * kPer + k + 1;
      best_before = before;
      best_in = in[k];
    }
    before += in[k];
  }
  if (best) atomicMax(&sh->bin, best);
  __syncthreads();
  const uint32_t last = sh->bin;
  __syncthreads();
  if (best && best == last) {
    sh->bin = kBins - last;
    sh->before = best_before;
    sh->inside = best_in;
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ Params q) {
  constexpr int kDrop = Logit<T>::kDrop;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const SampleArgs& p = q.a;
  Shared* sh = reinterpret_cast<Shared*>(smem_raw);
  T* x = reinterpret_cast<T*>(sh + 1);
  const int ctas = q.ctas, rank = static_cast<int>(cluster_ctarank()), row = blockIdx.x / ctas;
  const int lane = threadIdx.x & 31;
  const int slice = q.run * kThreads, base = rank * slice, n = max(0, min(slice, p.vocab - base));
  if (threadIdx.x < 64) sh->powers[threadIdx.x] = kPowers.at[threadIdx.x];
  for (int i = threadIdx.x; i < 9 * (kBins / 2); i += kThreads) (&sh->sum[0][0][0])[i] = 0;
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const float heat = p.temperatures ? __ldg(p.temperatures + row) : p.temperature;
  const int top_k = p.top_ks ? __ldg(p.top_ks + row) : p.top_k;
  const float top_p = p.top_ps ? __ldg(p.top_ps + row) : p.top_p;
  const float min_p = p.min_ps ? __ldg(p.min_ps + row) : p.min_p;

  // The row's part into shared memory; NaN becomes -inf.
  float largest;
  {
    using L = Logit<T>;
    const T* from = static_cast<const T*>(p.logits) + row * p.row_stride + base;
    constexpr int kVec = 16 / sizeof(T);
    const int whole = reinterpret_cast<uintptr_t>(from) % 16 ? 0 : n / kVec * kVec;
    uint32_t most = L::kLowest;
#pragma unroll 4
    for (int i = threadIdx.x * kVec; i < whole; i += kThreads * kVec) {
      uint4 w = __ldg(reinterpret_cast<const uint4*>(from + i));
      w = make_uint4(L::larger(w.x, L::kLowest), L::larger(w.y, L::kLowest), L::larger(w.z, L::kLowest),
                     L::larger(w.w, L::kLowest));
      most = L::larger(L::larger(L::larger(most, w.x), L::larger(w.y, w.z)), w.w);
      *reinterpret_cast<uint4*>(x + i) = w;
    }
    const float2 two = L::both(most);
    largest = fmaxf(two.x, two.y);
    for (int i = whole + threadIdx.x; i < slice; i += kThreads) {
      float v = i < n ? L::load(from[i]) : -INFINITY;
      v = v == v ? v : -INFINITY;
      largest = fmaxf(largest, v);
      x[i] = L::store(v);
    }
  }
  float m = block_reduce(largest, sh->scratch, [](float a, float b) { return fmaxf(a, b); });
  if (threadIdx.x == 0) sh->largest = m;
  cluster_sync();
  m = cluster_reduce(&sh->largest, ctas, -INFINITY, [](float a, float b) { return fmaxf(a, b); });

  const int first = threadIdx.x * q.run;  // of this thread's tokens
  if (m == -INFINITY) {
    if (rank == 0 && threadIdx.x == 0) {
      p.tokens[row] = -1;
      p.logprobs[row] = NAN;
    }
    cluster_sync();  // no CTA leaves while a peer reads from it
    return;
  }
  if (!(heat > 0.f) || min_p > 1.f) {  // (no w is above one: the first token alone is kept)
    uint32_t at = 0xffffffffu;
    for (int j = q.run - 1; j >= 0; --j)
      if (Logit<T>::load(x[first + j]) == m) at = base + first + j;
    at = block_reduce(at, sh->scratch, [](uint32_t a, uint32_t b) { return min(a, b); });
    if (threadIdx.x == 0) sh->first = at;
    cluster_sync();
    at = cluster_reduce(&sh->first, ctas, 0xffffffffu, [](uint32_t a, uint32_t b) { return min(a, b); });
    if (rank == 0 && threadIdx.x == 0) {
      p.tokens[row] = at;
      p.logprobs[row] = 0.f;
    }
    cluster_sync();
    return;
  }
  if (m == INFINITY) {
    // Tokens at +inf weigh one and all others nothing, whatever the temperature.
    for (int i = threadIdx.x; i < slice; i += kThreads)
      x[i] = Logit<T>::store(Logit<T>::load(x[i]) == INFINITY ? 0.f : -INFINITY);
    largest = largest == INFINITY ? 0.f : -INFINITY;
    m = 0.f;
    __syncthreads();
  }
  const double per_t = 1.4426950408889634 / fmax(static_cast<double>(heat), 1e-37);
  Weights weight{m, static_cast<float>(per_t), 0.f, sh->powers};
  weight.low = static_cast<float>(per_t - weight.high);

  const u64 least_w = min_p > 0.f ? static_cast<u64>(ceil(static_cast<double>(min_p) * 17592186044416.0)) : 0;
  // The token is the first whose running sum exceeds this integer: u total, held
  // below total.
  const float u = fmaxf(__ldg(p.uniform + row), 0.f);
  auto goal_of = [&](u64 total) {
    const u64 goal = static_cast<u64>(fmin(static_cast<double>(u) * static_cast<double>(total), 9.0e18));
    return goal < total ? goal : total - 1;
  };

  // Kept: logits above `cut`, and the first `room` of those at it (or all).
  float cut = -INFINITY;
  uint32_t room = 0;
  bool all_at = true;
  bool listed = false;  // the tokens that a cut may fall on are in the list
  int round = 0;
  auto each = [&](auto f) {
    if (listed) {
      for (int i = threadIdx.x, c = sh->listed; i < c; i += kThreads) f(Logit<T>::load(x[sh->list[i]]));
    } else {
      each_word<T, false>(x, threadIdx.x, kThreads, n, [&](float v, int) { f(v); });
    }
  };
  // Lists this CTA's tokens from `least` on; a list that they do not fit is not used.
  // (A second list is made where they did not fit the first; the peers have read its
  // length by the cluster's barrier between.)
  auto make_list = [&](float least) {
    if (threadIdx.x == 0) sh->listed = 0;
    __syncthreads();
    // (Counted first, so that a warp takes its places in the list at once.)
    uint32_t c = 0;
    each_word<T, true>(x, threadIdx.x, kThreads, slice, [&](float v, int) { c += v >= least; });
    uint32_t sum = c, at = 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += t;
    }
    if (lane == 31) at = atomicAdd(&sh->listed, sum);
    at = __shfl_sync(0xffffffffu, at, 31) + sum - c;
    if (c && at + c <= kListed)
      each_word<T, true>(x, threadIdx.x, kThreads, slice, [&](float v, int i) {
        if (v >= least) sh->list[at++] = static_cast<uint16_t>(i);
      });
    __syncthreads();
    listed = sh->listed <= kListed;
  };
  // Where the row's lists hold kDirect tokens at most, the first CTA ranks them
  // by comparing each with all, and draws: whether that was done. top_k counts
  // where `sum` (over what top-k keeps) is not known yet.
  auto draw_listed = [&](u64 sum) {
    cluster_sync();
    uint32_t before;
    const uint32_t c = cluster_reduce(&sh->listed, ctas, 0u, [](uint32_t a, uint32_t b) { return a + b; }, rank, &before);
    if (c > kDirect) return false;
    Ranked* all = reinterpret_cast<Ranked*>(&sh->own[0][0]);
    Ranks* half = reinterpret_cast<Ranks*>(all + kDirect);
    static_assert(kDirect * (sizeof(Ranked) + sizeof(Ranks)) <= sizeof(sh->own), "lists");
    for (uint32_t i = threadIdx.x; i < sh->listed; i += kThreads) {
      const int place = sh->list[i];
      const float v = Logit<T>::load(x[place]);
      const uint32_t to = map_to_rank(all + before + i, 0);
      asm volatile("st.shared::cluster.v2.b64 [%0], {%1, %2};" ::"r"(to), "l"(weight(v)),
                   "l"(static_cast<u64>(base + place) << 32 | __float_as_uint(v))
                   : "memory");
    }
    cluster_sync();
    if (rank > 0) return true;
    // A token's half of the others, by two threads each.
    const uint32_t me = threadIdx.x & (kDirect - 1), from = threadIdx.x >= kDirect ? c / 2 : 0;
    const uint32_t to = threadIdx.x >= kDirect ? c : c / 2;
    const Ranked mine = all[me < c ? me : 0];
    Ranks r{0, 0, 0};
    if (me < c)
      for (uint32_t j = from; j < to; ++j) {
        const Ranked t = all[j];
        r.w += t.v > mine.v ? t.w : 0;
        r.greater += t.v > mine.v;
        r.ties += t.v == mine.v && t.place < mine.place;
      }
    if (threadIdx.x >= kDirect) half[me] = r;
    __syncthreads();
    const bool in = threadIdx.x < c;  // (of the first half of the threads: a token each)
    if (in) {
      r.w += half[me].w;
      r.greater += half[me].greater;
      r.ties += half[me].ties;
    }
    const auto plus = [](u64 a, u64 b) { return a + b; };
    const u64 ahead = r.w + r.ties * mine.w;  // the sum ranked before it
    bool keep = in && (sum > 0 || r.greater + r.ties < static_cast<uint32_t>(top_k));
    if (sum == 0) sum = block_reduce(keep ? mine.w : 0, sh->scratch, plus);
    if (top_p < 1.f)
      keep &= r.greater + r.ties == 0 || static_cast<double>(ahead) < static_cast<double>(top_p) * static_cast<double>(sum);
    keep &= mine.w >= least_w;
    const u64 w = keep ? mine.w : 0;
    const u64 total = block_reduce(w, sh->scratch, plus);
    if (threadIdx.x < kDirect) all[me] = Ranked{w, mine.v, in ? mine.place : 0xffffffffu};
    __syncthreads();
    // Running sums in the order of the places.
    u64 upto = 0;
    if (me < c)
      for (uint32_t j = from; j < to; ++j) upto += all[j].place <= mine.place ? all[j].w : 0;
    if (threadIdx.x >= kDirect) half[me].w = upto;
    __syncthreads();
    if (w) {
      upto += half[me].w;
      const u64 goal = goal_of(total);
      if (goal < upto && upto - w <= goal) {
        p.tokens[row] = mine.place;
        p.logprobs[row] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(total)));
      }
    }
    return true;
  };
  // Finds the key where take(sum before) is last true among those from `low`
  // up to the largest; leaves the sums before it and at it.
  auto search = [&](auto weighed, uint32_t low, auto add, auto take, u64* before, u64* inside) {
    uint32_t high = key_of<kDrop>(m);
    *before = 0;
    while (true) {
      int shift = 0;
      while ((high - low) >> shift >= kBins) ++shift;
      search_round<decltype(weighed)::value>(sh, round, ctas, [&] {
        each([&](float v) {
          const uint32_t key = key_of<kDrop>(v);
          if (key >= low && key <= high) add(v, &sh->own[0][(key - low) >> shift]);
        });
      }, [&](u64 in) { return take(*before + in); });
      ++round;
      *before += sh->before;
      *inside = sh->inside;
      low += sh->bin << shift;
      if (shift == 0) break;
      high = min(high, low + (1u << shift) - 1);
      __syncthreads();  // before the next round's bin
    }
    __syncthreads();
    return low;
  };
  if (top_k > 0 && top_k < p.vocab) {
    float least = -INFINITY;
    if (top_k <= ctas * kThreads) {
      // A histogram of the threads' maxima, down to an eighth of the largest
      // (or eight times it, below zero): at least k of them, and so of all
      // tokens, are not below where the k-th one's bin begins.
      const uint32_t low = key_of<kDrop>(m > 0.f ? m * 0.125f : m * 8.f), high = key_of<kDrop>(m);
      int shift = 0;
      while ((high - low) >> shift >= kBins) ++shift;
      search_round<false>(sh, round, ctas, [&] {
        const uint32_t key = key_of<kDrop>(largest);
        atomicAdd(&sh->own[0][key > low ? (key - low) >> shift : 0], 1u);
      }, [&](u64 before) { return before < static_cast<u64>(top_k); });
      ++round;
      if (sh->bin) least = value_of<kDrop>(low + (sh->bin << shift));
      __syncthreads();
    }
    if (least > -INFINITY) {
      make_list(least);
      if (draw_listed(0)) {
        cluster_sync();
        return;
      }
    }
    u64 before, inside;
    cut = value_of<kDrop>(search(std::false_type(), key_of<kDrop>(least), [](float, uint32_t* bin) { atomicAdd(bin, 1u); },
                                 [&](u64 ahead) { return ahead < static_cast<u64>(top_k); }, &before, &inside));
    room = static_cast<uint32_t>(top_k - before);
    all_at = room == inside;
  }
  if (top_p < 1.f) {
    // The sum over what top-k keeps (all of those at its cut first), the sums
    // above five weights, and the number of those at the cut.
    u64 sums[kLevels + 2] = {};
    const auto plus = [](u64 a, u64 b) { return a + b; };
    auto take = [&](float v) {
      const u64 w = v >= cut ? weight(v) : 0;
      sums[kLevels] += w;
      sums[kLevels + 1] += v == cut;
#pragma unroll
      for (int k = 0; k < kLevels; ++k)
        if (w >= u64(1) << (40 - 3 * k)) sums[k] += w;
    };
    if (listed) {
      each(take);
    } else {
      each_word<T, true>(x, threadIdx.x, kThreads, slice, [&](float v, int) { take(v); });
    }
#pragma unroll
    for (int k = 0; k < kLevels + 2; ++k) {
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) sums[k] += __shfl_xor_sync(0xffffffffu, sums[k], off);
      if (lane == 0) sh->wide[k][threadIdx.x >> 5] = sums[k];
    }
    __syncthreads();
    if (threadIdx.x < 32 * (kLevels + 2)) {
      u64 v = lane < kWarps ? sh->wide[threadIdx.x >> 5][lane] : 0;
#pragma unroll
      for (int off = kWarps / 2; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      if (lane == 0) sh->parts[threadIdx.x >> 5] = v;
    }
    cluster_sync();
#pragma unroll
    for (int k = 0; k < kLevels + 2; ++k) sums[k] = cluster_reduce(&sh->parts[k], ctas, u64(0), plus);
    const u64 left_out = all_at ? 0 : (sums[kLevels + 1] - room) * weight(cut);
    const double target = static_cast<double>(top_p) * static_cast<double>(sums[kLevels] - left_out);
    // From here on the search begins: the same in all CTAs, whether their tokens
    // are listed or not. Some room for the rounding of the logit that goes with a
    // weight.
    float least = cut;
#pragma unroll
    for (int k = kLevels - 1; k >= 0; --k)
      if (static_cast<double>(sums[k]) >= target)
        least = fmaxf(cut, m - heat * (0.6931472f * 1.0001f) * (3 * k + 4) - fabsf(m) * 1e-5f);
    if (least > cut) {
      if (!listed) make_list(least);
      // (Behind a top-k that is not the whole row's its ties would count too.)
      if (cut == -INFINITY && draw_listed(sums[kLevels])) {
        cluster_sync();
        return;
      }
    }
    u64 before, inside;
    const float low = value_of<kDrop>(search(std::true_type(), key_of<kDrop>(least), [&](float v, uint32_t* bin) {
      const u64 w = weight(v);
      if (const uint32_t part = static_cast<uint32_t>(w) & 0xffffu) atomicAdd(bin, part);
      if (const uint32_t part = static_cast<uint32_t>(w >> 16) & 0xffffu) atomicAdd(bin + kBins, part);
      if (const uint32_t part = static_cast<uint32_t>(w >> 32)) atomicAdd(bin + 2 * kBins, part);
    }, [&](u64 ahead) { return ahead == 0 || static_cast<double>(ahead) < target; }, &before, &inside));
    // All tokens at this logit weigh the same: of them those that have less than
    // the target before them, and one at least where nothing is before.
    const u64 w = weight(low);
    const double per = 1.0 / static_cast<double>(w), most = (target - static_cast<double>(before)) * per;
    const u64 at_low = static_cast<u64>(static_cast<double>(inside) * per + 0.5);  // (below 2^18: exact)
    const u64 here = low == cut && !all_at ? room : at_low;
    u64 few = most >= static_cast<double>(here) ? here : (most < 0.0 ? 0 : static_cast<u64>(most));
    while (few < here && static_cast<double>(before + few * w) < target) ++few;
    while (few > 0 && !(static_cast<double>(before + (few - 1) * w) < target)) --few;
    if (before == 0 && few == 0) few = 1;
    cut = low;
    room = static_cast<uint32_t>(few);
    all_at = few == at_low;
  }

  // Where not all tokens at the cut are kept: the place of the last one that is.
  int limit = slice;
  if (!all_at) {
    uint32_t ties = 0;
    if (listed) {
      for (int i = threadIdx.x; i < kThreads; i += kThreads) sh->own[0][i] = 0;
      __syncthreads();
      for (int i = threadIdx.x, c = sh->listed; i < c; i += kThreads)
        if (Logit<T>::load(x[sh->list[i]]) == cut) atomicAdd(&sh->own[0][sh->list[i] / q.run], 1u);
      __syncthreads();
      ties = sh->own[0][threadIdx.x];
    } else {
      each_word<T, true>(x + first, 0, 1, q.run, [&](float v, int) { ties += v == cut; });
    }
    u64 all;
    uint32_t ahead = static_cast<uint32_t>(block_scan(ties, sh->scratch, &all)), before;
    if (threadIdx.x == 0) sh->cut_ties = static_cast<uint32_t>(all);
    cluster_sync();
    cluster_reduce(&sh->cut_ties, ctas, 0u, [](uint32_t a, uint32_t b) { return a + b; }, rank, &before);
    ahead += before;
    if (threadIdx.x == 0) sh->limit = before < room ? slice : -1;
    __syncthreads();
    if (ahead < room && room < ahead + ties) {
      uint32_t left = room - ahead;
      for (int j = 0; left > 0; ++j)
        if (Logit<T>::load(x[first + j]) == cut && --left == 0) sh->limit = first + j;
    } else if (ahead == room && ties > 0 && ahead > before) {
      // The last one kept lies in an earlier run of this CTA, which ends with it.
      atomicMin(&sh->limit, first - 1);
    }
    __syncthreads();
    limit = sh->limit;
  }
  // W of a token, by its place, if it is kept.
  auto kept = [&](float v, int place) -> u64 {
    if (v < cut || (v == cut && place > limit)) return 0;
    const u64 w = weight(v);
    return w >= least_w ? w : 0;
  };
  u64 mine = 0, total = 0;
  if (cut == -INFINITY) {
    each_word<T, true>(x + first, 0, 1, q.run, [&](float v, int) {
      const u64 w = weight(v);
      mine += w >= least_w ? w : 0;
    });
  } else if (listed) {
    // From the list: a run's sum in 16 bits of the weights each.
    for (int i = threadIdx.x; i < 3 * kThreads; i += kThreads) (&sh->own[0][0])[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x, c = sh->listed; i < c; i += kThreads) {
      const int place = sh->list[i];
      const u64 w = kept(Logit<T>::load(x[place]), place);
      uint32_t* run = &sh->own[0][place / q.run];
      if (const uint32_t part = static_cast<uint32_t>(w) & 0xffffu) atomicAdd(run, part);
      if (const uint32_t part = static_cast<uint32_t>(w >> 16) & 0xffffu) atomicAdd(run + kThreads, part);
      if (const uint32_t part = static_cast<uint32_t>(w >> 32)) atomicAdd(run + 2 * kThreads, part);
    }
    __syncthreads();
    const uint32_t* run = &sh->own[0][threadIdx.x];
    mine = run[0] + (static_cast<u64>(run[kThreads]) << 16) + (static_cast<u64>(run[2 * kThreads]) << 32);
  } else {
    each_word<T, true>(x + first, 0, 1, q.run, [&](float v, int j) { mine += kept(v, first + j); });
  }
  u64 before = block_scan(mine, sh->scratch, &total);
  if (threadIdx.x == 0) sh->total = total;
  cluster_sync();
  {
    u64 ahead_of;
    total = cluster_reduce(&sh->total, ctas, u64(0), [](u64 a, u64 b) { return a + b; }, rank, &ahead_of);
    before += ahead_of;
  }
  const u64 goal = goal_of(total);
  const unsigned found = __ballot_sync(0xffffffffu, before <= goal && goal < before + mine);
  if (found) {
    // The warp looks through the one thread's tokens, 32 at a time.
    const int src = __ffs(found) - 1;
    before = __shfl_sync(0xffffffffu, before, src);
    const int from = __shfl_sync(0xffffffffu, first, src);
    for (int j0 = 0; j0 < q.run; j0 += 32) {
      const float v = j0 + lane < q.run ? Logit<T>::load(x[from + j0 + lane]) : -INFINITY;
      const u64 w = kept(v, from + j0 + lane);
      u64 sum = w;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += t;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + sum > goal);
      if (past) {
        if (lane == __ffs(past) - 1) {
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
  // CTAs a row: enough for 64 KB of it each at most, so that two CTAs share an
  // SM, and, while they do not fill the GPU, until a CTA has 2048 tokens.
  constexpr int kPack = 4 / sizeof(T), kMost = 16384 * kPack;
  int ctas = 1;
  while (ctas < kMaxCtas && (a.vocab > ctas * kMost || (static_cast<int64_t>(a.rows) * ctas <= num_sms &&
                                                        a.vocab > ctas * 2048)))
    ctas *= 2;
  p.ctas = ctas;
  p.run = kPack * (((a.vocab + ctas - 1) / ctas + kPack * kThreads - 1) / (kPack * kThreads) | 1);
  const size_t smem = sizeof(Shared) + static_cast<size_t>(p.run) * kThreads * sizeof(T);
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
