// Rotation and storing of a batch of tokens' queries, keys and values: one
// pass over the QKV projection's rows that norms the query and key heads
// (optional), rotates them by their positions and writes queries to a dense
// tensor and keys and values into their pages. No reference counterpart: the
// reference only models the cache's bytes (dequant/byte_model.py:214-219).
//
//   y     = x * rsqrt(mean(x^2) + eps) * w           (with a norm; per head)
//   (a,b) = (y_i, y_j),  j = i + R/2  or  (i, j) = (2p, 2p + 1)
//   a'    = a cos - b sin,  b' = b cos + a sin       (first R values; the rest pass)
//
// in fp32 with one rounding at the end; cos and sin come from a table of
// positions, so every scaling of the frequencies is the caller's.
//
// Bound by HBM: each row is read once and each head written once. A group of
// D / 16 lanes holds a head, and a lane two runs of eight values: in the half
// layout those at i and i + R/2, so that both values of a rotated pair lie in
// one lane and share a table entry; interleaved pairs lie in one lane anyway.
// A warp takes a few heads of one token, whose table entries stay in
// registers; the sum of squares is one shuffle reduction. What it measured
// (B200, 8192 tokens of 64 + 2 x 8 heads of 128, bf16, norms): 62.5 us a call,
// 5.4 TB/s of the 6.4 that a copy reaches (58.5 us and 5.8 replayed from a graph,
// which the following figures are). Registers and stores decide: 128 registers
// (two blocks of 256 an SM) 79 us, 80 (three) 69; with stores that do not stay
// in the L2 cache 62, in blocks of 128 threads 59. Runs of four values instead
// of eight (more, narrower accesses) 84 us; one head a lane group at a time 84.
#include <cstdint>

#include "paged.cuh"

namespace dqg {
namespace {

constexpr int kThreads = 128;
constexpr int kIter = 4;  // heads a lane group takes one after the other

template <typename E>
struct AppendParams {
  const E* qkv;
  const float* cosv;
  const float* sinv;
  const int64_t* positions;
  const int64_t* slots;
  const E* q_norm;
  const E* k_norm;
  E* q_out;
  E* k;
  E* v;
  int64_t qkv_stride, n_positions, n_slots, page_stride, head_stride, row_stride;
  int T, hq, hkv, rot, page_shift, chunks;
  float eps;
};

enum Layout {
  kHalf,         // pairs (i, i + R/2), R a multiple of 16
  kInterleaved,  // pairs (2i, 2i + 1)
  kUneven        // pairs (i, i + R/2), any R: partners are read again from memory
};

template <typename E>
__device__ __forceinline__ void unpack8(uint4 v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = Elem<E>::unpack(w[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <typename E>
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(Elem<E>::pack(f[0], f[1]), Elem<E>::pack(f[2], f[3]), Elem<E>::pack(f[4], f[5]),
                    Elem<E>::pack(f[6], f[7]));
}

template <typename E, int D, int ITER, int LAYOUT>
__global__ void __launch_bounds__(kThreads, LAYOUT == kUneven ? 4 : 5)
    paged_append_kernel(const __grid_constant__ AppendParams<E> p) {
  constexpr int kLanes = D / 16;        // lanes a head
  constexpr int kGroups = 32 / kLanes;  // heads a warp holds at a time
  const int64_t w = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t token = w / p.chunks;
  const int chunk = static_cast<int>(w - token * p.chunks);
  const int lane = threadIdx.x & 31, c = lane % kLanes, grp = lane / kLanes;
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  if (token >= p.T) return;
  const int rotated = p.hq + p.hkv, n_heads = rotated + p.hkv;
  const int h0 = chunk * ITER * kGroups + grp;
  // The lane's two runs of eight values. Half layout: the first R / 16 lanes
  // hold the pairs, the others what passes.
  const int rc = p.rot / 16;
  const bool pairs = LAYOUT != kHalf || c < rc;
  const int ea = LAYOUT == kHalf ? (pairs ? 8 * c : 16 * c) : 16 * c;
  const int eb = LAYOUT == kHalf && pairs ? ea + p.rot / 2 : ea + 8;
  const E* row = p.qkv + token * p.qkv_stride;
  uint4 xa[ITER], xb[ITER];
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int h = h0 + it * kGroups;
    if (h < n_heads) {
      xa[it] = __ldcs(reinterpret_cast<const uint4*>(row + static_cast<int64_t>(h) * D + ea));
      xb[it] = __ldcs(reinterpret_cast<const uint4*>(row + static_cast<int64_t>(h) * D + eb));
    }
  }
  int64_t pos = __ldg(p.positions + token);
  int64_t slot = __ldg(p.slots + token);
  if (pos < 0 || pos >= p.n_positions || slot >= p.n_slots) {
    if (lane == 0) atomicOr(&g_status, kStatusBadIndex);
    pos = pos < 0 ? 0 : (pos >= p.n_positions ? p.n_positions - 1 : pos);
    if (slot >= p.n_slots) slot = -1;
  }
  const int half = p.rot / 2;
  // Table entries of the lane's eight pairs (uneven: of its sixteen values).
  constexpr int kTab = LAYOUT == kUneven ? 16 : 8;
  float cs[kTab], sn[kTab];
  if (h0 - grp < rotated) {
    const float* cr = p.cosv + pos * half;
    const float* sr = p.sinv + pos * half;
#pragma unroll
    for (int e = 0; e < kTab; ++e) {
      const int i = LAYOUT == kUneven ? (ea + e < half ? ea + e : ea + e - half) : 8 * c + e;
      const bool in = LAYOUT == kUneven ? ea + e < p.rot : i < half;
      cs[e] = in ? __ldg(cr + i) : 1.f;
      sn[e] = in ? __ldg(sr + i) : 0.f;
    }
  }
  const int64_t page = slot >> p.page_shift;
  const int64_t place = slot & ((int64_t(1) << p.page_shift) - 1);
  const int64_t base = page * p.page_stride + place * p.row_stride;
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int h = h0 + it * kGroups;
    const bool is_k = h >= p.hq;
    // (Warp-uniform: the shuffles below are taken by the whole warp.)
    if (h - grp < rotated) {
      float a[8], b[8];
      unpack8<E>(h < n_heads ? xa[it] : make_uint4(0u, 0u, 0u, 0u), a);
      unpack8<E>(h < n_heads ? xb[it] : make_uint4(0u, 0u, 0u, 0u), b);
      float r = 1.f;
      if (p.q_norm) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(a[e], a[e], fmaf(b[e], b[e], ss));
#pragma unroll
        for (int off = kLanes / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
        r = rsqrtf(fmaf(ss, 1.f / D, p.eps));
        float wa[8], wb[8];
        const E* nw = is_k ? p.k_norm : p.q_norm;
        unpack8<E>(__ldg(reinterpret_cast<const uint4*>(nw + ea)), wa);
        unpack8<E>(__ldg(reinterpret_cast<const uint4*>(nw + eb)), wb);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[e] *= r * wa[e];
          b[e] *= r * wb[e];
        }
      }
      if (h < rotated) {
        if (LAYOUT == kHalf) {
          if (pairs) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float x = a[e], y = b[e];
              a[e] = fmaf(x, cs[e], -(y * sn[e]));
              b[e] = fmaf(y, cs[e], x * sn[e]);
            }
          }
        } else if (LAYOUT == kInterleaved) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float* t = e < 4 ? a + 2 * e : b + 2 * (e - 4);
            if (8 * c + e < half) {
              const float x = t[0], y = t[1];
              t[0] = fmaf(x, cs[e], -(y * sn[e]));
              t[1] = fmaf(y, cs[e], x * sn[e]);
            }
          }
        } else {
          const E* head = row + static_cast<int64_t>(h) * D;
          const E* nw = is_k ? p.k_norm : p.q_norm;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int i = ea + e, j = i < half ? i + half : i - half;
            float* t = e < 8 ? a + e : b + e - 8;
            if (i < p.rot) {
              float y = Elem<E>::load(head + j);
              if (p.q_norm) y *= r * Elem<E>::load(nw + j);
              *t = fmaf(*t, cs[e % kTab], i < half ? -(y * sn[e % kTab]) : y * sn[e % kTab]);
            }
          }
        }
        xa[it] = pack8<E>(a);
        xb[it] = pack8<E>(b);
      }
    }
    if (h >= n_heads) continue;
    E* dst;
    if (!is_k) {
      dst = p.q_out + (token * p.hq + h) * D;
    } else {
      if (slot < 0) continue;
      dst = h < rotated ? p.k + base + (h - p.hq) * p.head_stride : p.v + base + (h - rotated) * p.head_stride;
    }
    __stcs(reinterpret_cast<uint4*>(dst + ea), xa[it]);
    __stcs(reinterpret_cast<uint4*>(dst + eb), xb[it]);
  }
}

template <typename E, int D, int ITER>
cudaError_t launch(const PagedPool& pool, const AppendArgs& a, cudaStream_t stream) {
  AppendParams<E> p;
  p.qkv = static_cast<const E*>(a.qkv);
  p.cosv = a.cosv;
  p.sinv = a.sinv;
  p.positions = a.positions;
  p.slots = a.slots;
  p.q_norm = static_cast<const E*>(a.q_norm);
  p.k_norm = static_cast<const E*>(a.k_norm);
  p.q_out = static_cast<E*>(a.q_out);
  p.k = static_cast<E*>(const_cast<void*>(pool.k));
  p.v = static_cast<E*>(const_cast<void*>(pool.v));
  p.qkv_stride = a.qkv_stride;
  p.n_positions = a.n_positions;
  p.n_slots = pool.n_pages * pool.page_size;
  p.page_stride = pool.page_stride;
  p.head_stride = pool.head_stride;
  p.row_stride = pool.row_stride;
  p.T = a.T;
  p.hq = a.hq;
  p.hkv = pool.n_kv_heads;
  p.rot = a.rot;
  p.page_shift = 0;
  while ((1 << p.page_shift) < pool.page_size) ++p.page_shift;
  p.eps = a.eps;
  constexpr int kPer = ITER * 32 / (D / 16);
  p.chunks = (a.hq + 2 * pool.n_kv_heads + kPer - 1) / kPer;
  const int64_t warps = static_cast<int64_t>(a.T) * p.chunks;
  const int64_t blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
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
  if (a.interleaved) return cudaLaunchKernelEx(&cfg, paged_append_kernel<E, D, ITER, kInterleaved>, p);
  if (a.rot % 16 == 0) return cudaLaunchKernelEx(&cfg, paged_append_kernel<E, D, ITER, kHalf>, p);
  return cudaLaunchKernelEx(&cfg, paged_append_kernel<E, D, ITER, kUneven>, p);
}

template <typename E, int D>
cudaError_t launch_iter(const PagedPool& pool, const AppendArgs& a, int num_sms,
                        cudaStream_t stream) {
  // kIter heads a lane group once that still fills the GPU's warps; below it
  // one, so that a few tokens spread over the SMs.
  const int64_t groups = static_cast<int64_t>(a.T) * (a.hq + 2 * pool.n_kv_heads) * (D / 16) / 32;
  if (groups >= kIter * 64 * static_cast<int64_t>(num_sms)) return launch<E, D, kIter>(pool, a, stream);
  return launch<E, D, 1>(pool, a, stream);
}

}  // namespace

cudaError_t launch_paged_append(const PagedPool& pool, const AppendArgs& a, int num_sms,
                                cudaStream_t stream) {
  if (pool.bf16)
    return pool.D == 128 ? launch_iter<__nv_bfloat16, 128>(pool, a, num_sms, stream)
                         : launch_iter<__nv_bfloat16, 64>(pool, a, num_sms, stream);
  return pool.D == 128 ? launch_iter<__half, 128>(pool, a, num_sms, stream)
                       : launch_iter<__half, 64>(pool, a, num_sms, stream);
}

}  // namespace dqg

DQG_STATUS_READER(read_status_append)
