// The draw of one token from each row of logits. No reference counterpart.
//
//   w_i = exp((l_i - max l) / T),  W_i = round(2^44 w_i)
//   kept: rank(i) < top_k, sum of W ranked before < top_p * sum over top_k, w_i >= min_p
//   token = first i, by index, with (sum of kept W up to i) > u * (their sum)
//
// Ranks are by logit, the lower index first. All sums are of 64-bit integers:
// exact, so that neither the order of summation nor the number of threads or
// CTAs changes a token. A W is exact to about 2^-31 of itself: the exponent is
// formed in pairs of fp32 numbers, its fraction in 64ths from a table and the rest
// by a polynomial (a 64-bit exp took more than half of the time).
//
// A cluster of up to eight CTAs takes a row; each holds a part of it in shared
// memory, and a thread a run of consecutive tokens of that. The logit at which
// top-k or top-p cuts is found from histograms of the ordered bits of the
// logits (numbers, or weights), 1024 bins of equal width at a time, until a bin
// is one logit: a CTA's own histogram first, whose bins in use are then added to
// a sum that every CTA has, so that one barrier of the cluster is enough. What
// lies far below a cut stays out of the histograms: top-k's cut is above what
// the k-th largest of the threads' maxima is above, and top-p's above the
// largest of four weights that has top_p of the sum above it. The tokens that
// are left, mostly a few, are listed once and read from there.
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
constexpr int kListed = 2048;           // tokens that a CTA's list holds
constexpr int kLevels = 4;              // weights 2^-4, 2^-8, 2^-12, 2^-16
constexpr u64 kOne = u64(1) << 44;

struct Params {
  SampleArgs a;
  int ctas;  // a row
  int run;   // tokens a thread: odd, so that reads of shared memory do not conflict
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

template <typename T>
struct Logit;
template <>
struct Logit<float> {
  static constexpr int kDrop = 0;  // low bits of an fp32 value that these never use
  static __device__ __forceinline__ float load(float v) { return v; }
};
template <>
struct Logit<__half> {
  static constexpr int kDrop = 13;
  static __device__ __forceinline__ float load(__half v) { return __half2float(v); }
};
template <>
struct Logit<__nv_bfloat16> {
  static constexpr int kDrop = 16;
  static __device__ __forceinline__ float load(__nv_bfloat16 v) { return __bfloat162float(v); }
};

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

struct Shared {
  Power powers[64];
  uint32_t own[3][kBins];     // this CTA's histogram: numbers, or 16 bits of the weights each
  uint32_t sum[2][3][kBins];  // the cluster's, in turn: numbers, or 24 bits of the weights each
  float list[kListed];
  u64 scratch[kWarps];
  u64 parts[kLevels + 1];     // of sums, read by the peers
  float largest;
  uint32_t first, ties, cut_ties, listed;
  u64 total;
  uint32_t bin;               // of the cut
  u64 before, inside;         // ahead of it, and in it
};

struct Weights {
  float m, high, low;  // the largest logit; log2(e) / T in two parts
  bool inf;            // m is +inf
  const Power* powers;
  // W of a logit.
  __device__ __forceinline__ u64 operator()(float v) const {
    if (inf) return v == INFINITY ? kOne : 0;
    // s + err = v - m and p + e = (v - m) log2(e) / T, in twice the precision.
    const float s = v - m, back = s - v;
    const float p = s * high;
    if (!(p >= -46.f)) return 0;
    const float err = (v - (s - back)) + (-m - back);
    const float e = fmaf(err, high, fmaf(s, low, fmaf(s, high, -p)));
    const float t = fmaf(p, 64.f, 12582912.f);  // 1.5 * 2^23: the fraction's last bit is one
    const int n = __float_as_int(t) - 0x4b400000;
    const float r = fmaf(t - 12582912.f, -1.f / 64.f, p) + e;  // 64ths out; at most 1/128
    // 2^r - 1
    const float q = r * fmaf(r, fmaf(r, fmaf(r, 9.6181291e-3f, 5.5504109e-2f), 2.4022651e-1f), 6.9314718e-1f);
    const Power w = powers[n & 63];
    const u64 one = w.fixed + (static_cast<long long>(__float2int_rn(q * w.scaled)) << 13);
    const int down = -(n >> 6);
    return down ? (one + (u64(1) << (down - 1))) >> down : one;
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
// sh->before and sh->inside. The buffers of sh->sum take turns; the next
// round's is zeroed here.
template <bool kWeighed, class Add, class Take>
__device__ __forceinline__ void search_round(Shared* sh, int turn, int ctas, Add add, Take take) {
  constexpr int kArrays = kWeighed ? 3 : 1;
  for (int i = threadIdx.x; i < kArrays * kBins; i += kThreads) (&sh->own[0][0])[i] = 0;
  for (int i = threadIdx.x; i < 3 * kBins; i += kThreads) (&sh->sum[turn ^ 1][0][0])[i] = 0;
  if (threadIdx.x == 0) sh->bin = 0;
  __syncthreads();
  add();
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int bin = threadIdx.x + k * kThreads;
    if (kWeighed) {
      const u64 w = sh->own[0][bin] + (static_cast<u64>(sh->own[1][bin]) << 16) + (static_cast<u64>(sh->own[2][bin]) << 32);
      if (w == 0) continue;
      for (int r = 0; r < ctas; ++r)
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          const uint32_t part = static_cast<uint32_t>(w >> (24 * j)) & 0xffffffu;
          if (part) peer_add(&sh->sum[turn][j][bin], r, part);
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
    if (kWeighed) in[k] += (static_cast<u64>(sh->sum[turn][1][top - k]) << 24) + (static_cast<u64>(sh->sum[turn][2][top - k]) << 48);
    mine += in[k];
  }
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
  float* x = reinterpret_cast<float*>(sh + 1);
  const int ctas = q.ctas, rank = static_cast<int>(cluster_ctarank()), row = blockIdx.x / ctas;
  const int lane = threadIdx.x & 31;
  const int slice = q.run * kThreads, base = rank * slice, n = max(0, min(slice, p.vocab - base));
  if (threadIdx.x < 64) sh->powers[threadIdx.x] = kPowers.at[threadIdx.x];
  for (int i = threadIdx.x; i < 3 * kBins; i += kThreads) (&sh->sum[0][0][0])[i] = 0;
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
#pragma unroll 4
    for (int i = threadIdx.x * kVec; i < whole; i += kThreads * kVec) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(from + i));
      const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int k = 0; k < kVec; ++k) put(i + k, Logit<T>::load(v[k]));
    }
    for (int i = whole + threadIdx.x; i < n; i += kThreads) put(i, Logit<T>::load(from[i]));
    for (int i = n + threadIdx.x; i < slice; i += kThreads) x[i] = -INFINITY;
  }
  float m = block_reduce(largest, sh->scratch, [](float a, float b) { return fmaxf(a, b); });
  if (threadIdx.x == 0) {
    sh->largest = m;
    sh->listed = 0;
  }
  cluster_sync();
  for (int r = 0; r < ctas; ++r) m = fmaxf(m, peer(&sh->largest, r));

  const int first = threadIdx.x * q.run;  // of this thread's tokens
  if (m == -INFINITY) {
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
      for (int r = 1; r < ctas; ++r) at = min(at, peer(&sh->first, r));
      p.tokens[row] = at;
      p.logprobs[row] = 0.f;
    }
    cluster_sync();
    return;
  }
  const double per_t = 1.4426950408889634 / fmax(static_cast<double>(heat), 1e-37);
  Weights weight{m, static_cast<float>(per_t), 0.f, m == INFINITY, sh->powers};
  weight.low = static_cast<float>(per_t - weight.high);

  // Kept: logits above `cut`, and the first `room` of those at it (or all).
  float cut = -INFINITY;
  uint32_t room = 0;
  bool all_at = true;
  bool listed = false;  // the tokens that a cut may fall on are in the list
  int turn = 0;
  auto each = [&](auto f) {
    if (listed) {
      for (int i = threadIdx.x, c = sh->listed; i < c; i += kThreads) f(sh->list[i]);
    } else {
      for (int i = threadIdx.x; i < n; i += kThreads) f(x[i]);
    }
  };
  // Lists this CTA's tokens from `least` on; a list that they do not fit is not used.
  auto make_list = [&](float least) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = x[i];
      if (v < least) continue;
      const uint32_t at = atomicAdd(&sh->listed, 1u);
      if (at < kListed) sh->list[at] = v;
    }
    __syncthreads();
    listed = sh->listed <= kListed;
  };
  // Finds the key where take(sum before) is last true among those from `low`
  // up to the largest; leaves the sums before it and at it.
  auto search = [&](auto weighed, uint32_t low, auto add, auto take, u64* before, u64* inside) {
    uint32_t high = key_of<kDrop>(m);
    *before = 0;
    while (true) {
      int shift = 0;
      while ((high - low) >> shift >= kBins) ++shift;
      search_round<decltype(weighed)::value>(sh, turn, ctas, [&] {
        each([&](float v) {
          const uint32_t key = key_of<kDrop>(v);
          if (key >= low && key <= high) add(v, &sh->own[0][(key - low) >> shift]);
        });
      }, [&](u64 in) { return take(*before + in); });
      turn ^= 1;
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
      search_round<false>(sh, turn, ctas, [&] {
        const uint32_t key = key_of<kDrop>(largest);
        atomicAdd(&sh->own[0][key > low ? (key - low) >> shift : 0], 1u);
      }, [&](u64 before) { return before < static_cast<u64>(top_k); });
      turn ^= 1;
      if (sh->bin) least = value_of<kDrop>(low + (sh->bin << shift));
      __syncthreads();
    }
    if (least > -INFINITY) make_list(least);
    u64 before, inside;
    cut = value_of<kDrop>(search(std::false_type(), key_of<kDrop>(least), [](float, uint32_t* bin) { atomicAdd(bin, 1u); },
                                 [&](u64 ahead) { return ahead < static_cast<u64>(top_k); }, &before, &inside));
    room = static_cast<uint32_t>(top_k - before);
    all_at = room == inside;
  }
  if (top_p < 1.f) {
    // The sum over what top-k keeps (all of those at its cut first), and the
    // sums above four weights.
    u64 sums[kLevels + 1] = {};
    uint32_t ties = 0;
    each([&](float v) {
      if (v < cut) return;
      const u64 w = weight(v);
      ties += v == cut;
      sums[kLevels] += w;
#pragma unroll
      for (int k = 0; k < kLevels; ++k)
        if (w >= kOne >> (4 * k + 4)) sums[k] += w;
    });
    const u64 at_cut = cut > -INFINITY ? weight(cut) : 0;
#pragma unroll
    for (int k = 0; k <= kLevels; ++k) {
      const u64 t = block_reduce(sums[k], sh->scratch, [](u64 a, u64 b) { return a + b; });
      if (threadIdx.x == 0) sh->parts[k] = t;
    }
    ties = block_reduce(ties, sh->scratch, [](uint32_t a, uint32_t b) { return a + b; });
    if (threadIdx.x == 0) sh->ties = ties;
    cluster_sync();
    ties = 0;
#pragma unroll
    for (int k = 0; k <= kLevels; ++k) sums[k] = 0;
    for (int r = 0; r < ctas; ++r) {
#pragma unroll
      for (int k = 0; k <= kLevels; ++k) sums[k] += peer(&sh->parts[k], r);
      ties += peer(&sh->ties, r);
    }
    const u64 left_out = all_at ? 0 : (ties - room) * at_cut;
    const double target = static_cast<double>(top_p) * static_cast<double>(sums[kLevels] - left_out);
    float least = cut;
    if (!listed && !weight.inf) {
      // Some room for the rounding of the logit that goes with a weight.
#pragma unroll
      for (int k = kLevels - 1; k >= 0; --k)
        if (static_cast<double>(sums[k]) >= target)
          least = fmaxf(cut, m - heat * (2.7725887f * 1.0001f) * (k + 1) - fabsf(m) * 1e-5f);
      if (least > cut) make_list(least);
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
    const u64 here = low == cut && !all_at ? room : inside / w;
    const double most = (target - static_cast<double>(before)) / static_cast<double>(w);
    u64 few = most >= static_cast<double>(here) ? here : (most < 0.0 ? 0 : static_cast<u64>(most));
    while (few < here && static_cast<double>(before + few * w) < target) ++few;
    while (few > 0 && !(static_cast<double>(before + (few - 1) * w) < target)) --few;
    if (before == 0 && few == 0) few = 1;
    cut = low;
    room = static_cast<uint32_t>(few);
    all_at = few == inside / w;
  }

  // Tokens at the cut that this thread's come behind, where not all are kept.
  uint32_t ahead = 0;
  if (!all_at) {
    uint32_t ties = 0;
    for (int j = 0; j < q.run; ++j) ties += x[first + j] == cut;
    u64 all;
    ahead = static_cast<uint32_t>(block_scan(ties, sh->scratch, &all));
    if (threadIdx.x == 0) sh->cut_ties = static_cast<uint32_t>(all);
    cluster_sync();
    for (int i = 0; i < rank; ++i) ahead += peer(&sh->cut_ties, i);
  }
  // W of a token if it is kept; *tie: tokens at the cut before it.
  const u64 least_w = min_p > 0.f ? static_cast<u64>(ceil(static_cast<double>(min_p) * 17592186044416.0)) : 0;
  auto kept = [&](float v, uint32_t* tie) -> u64 {
    if (v < cut) return 0;
    if (v == cut && !all_at && (*tie)++ >= room) return 0;
    const u64 w = weight(v);
    return w >= least_w ? w : 0;
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
    const u64 t = peer(&sh->total, i);
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
      const unsigned at_cut = __ballot_sync(0xffffffffu, j0 + lane < q.run && v == cut);
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
