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
// D / 8 lanes holds a head, 16 bytes a lane, and a warp takes a few heads of
// one token, whose table entries then stay in registers; the partner of a
// rotated value lies in another lane's registers (half layout) or in the lane
// itself (interleaved), and the sum of squares is one shuffle reduction.
#include <cstdint>

#include "paged.cuh"

namespace dqg {
namespace {

constexpr int kThreads = 256;

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
  bool interleaved;
};

// ALIGNED: the half layout's partner values are whole lanes away (R a
// multiple of 16), or every pair lies in one lane (interleaved). Otherwise
// partners are read again from memory, one at a time.
template <typename E, int D, int ITER, bool ALIGNED>
__global__ void __launch_bounds__(kThreads)
    paged_append_kernel(const __grid_constant__ AppendParams<E> p) {
  constexpr int kLanes = D / 8;         // lanes a head
  constexpr int kGroups = 32 / kLanes;  // heads a warp holds at a time
  const int64_t w = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t token = w / p.chunks;
  const int chunk = static_cast<int>(w - token * p.chunks);
  const int lane = threadIdx.x & 31, c = lane % kLanes, grp = lane / kLanes;
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  if (token >= p.T) return;
  const int n_heads = p.hq + 2 * p.hkv;
  const int h0 = chunk * ITER * kGroups + grp;
  const E* row = p.qkv + token * p.qkv_stride + c * 8;
  uint4 x[ITER];
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int h = h0 + it * kGroups;
    if (h < n_heads) x[it] = *reinterpret_cast<const uint4*>(row + static_cast<int64_t>(h) * D);
  }
  int64_t pos = p.positions[token];
  int64_t slot = p.slots[token];
  if (pos < 0 || pos >= p.n_positions || slot >= p.n_slots) {
    if (lane == 0) atomicOr(&g_status, kStatusBadIndex);
    pos = pos < 0 ? 0 : (pos >= p.n_positions ? p.n_positions - 1 : pos);
    if (slot >= p.n_slots) slot = -1;
  }
  const int half = p.rot / 2;
  // This lane's table entries: the pair that element e belongs to, and the
  // sign of its partner's term.
  float cs[8], sn[8];
  const float* cr = p.cosv + pos * half;
  const float* sr = p.sinv + pos * half;
  if (h0 - grp < p.hq + p.hkv) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = c * 8 + e;
      cs[e] = 1.f;
      sn[e] = 0.f;
      if (i < p.rot) {
        const bool lo = p.interleaved ? (i & 1) == 0 : i < half;
        const int pair = p.interleaved ? i >> 1 : (lo ? i : i - half);
        cs[e] = __ldg(cr + pair);
        sn[e] = lo ? -__ldg(sr + pair) : __ldg(sr + pair);
      }
    }
  }
  const int64_t page = slot >> p.page_shift;
  const int64_t place = slot & ((int64_t(1) << p.page_shift) - 1);
  const int64_t base = page * p.page_stride + place * p.row_stride + c * 8;
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int h = h0 + it * kGroups;
    // A group's lanes hold one head and a warp's groups neighbouring ones: the
    // shuffles below are taken by the whole warp.
    const bool rotated = h < p.hq + p.hkv;
    const bool is_k = h >= p.hq;
    float f[8], o[8];
    const uint32_t* xw = reinterpret_cast<const uint32_t*>(&x[it]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 t = h < n_heads ? Elem<E>::unpack(xw[e]) : make_float2(0.f, 0.f);
      f[2 * e] = t.x;
      f[2 * e + 1] = t.y;
    }
    const E* nw = is_k ? p.k_norm : p.q_norm;
    float r = 1.f;
    if (p.q_norm) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
      for (int off = kLanes / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      r = rsqrtf(ss * (1.f / D) + p.eps);
      const uint4 wv = *reinterpret_cast<const uint4*>(nw + c * 8);
      const uint32_t* ww = reinterpret_cast<const uint32_t*>(&wv);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 t = Elem<E>::unpack(ww[e]);
        f[2 * e] *= r * t.x;
        f[2 * e + 1] *= r * t.y;
      }
    }
    if (ALIGNED && !p.interleaved) {
      // Lane c + half / 8 (or c - half / 8) of the group holds the partners.
      const int dist = half >> 3;
      const int src = c * 8 < half ? c + dist : (c * 8 < p.rot ? c - dist : c);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = __shfl_sync(0xffffffffu, f[e], src, kLanes);
    } else if (p.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = f[e ^ 1];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = c * 8 + e;
        o[e] = 0.f;
        if (rotated && i < p.rot) {
          const int j = i < half ? i + half : i - half;
          o[e] = Elem<E>::load(row + static_cast<int64_t>(h) * D - c * 8 + j);
          if (p.q_norm) o[e] *= r * Elem<E>::load(nw + j);
        }
      }
    }
    if (h >= n_heads) continue;
    uint4 y = x[it];
    if (rotated) {
      uint32_t* yw = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c * 8 + e < p.rot) f[e] = fmaf(o[e], sn[e], f[e] * cs[e]);
#pragma unroll
      for (int e = 0; e < 4; ++e) yw[e] = Elem<E>::pack(f[2 * e], f[2 * e + 1]);
    }
    if (!is_k) {
      *reinterpret_cast<uint4*>(p.q_out + (token * p.hq + h) * D + c * 8) = y;
    } else if (slot >= 0) {
      const int kh = rotated ? h - p.hq : h - p.hq - p.hkv;
      *reinterpret_cast<uint4*>((rotated ? p.k : p.v) + base + kh * p.head_stride) = y;
    }
  }
}

template <typename E, int D, int ITER>
cudaError_t launch(const PagedPool& pool, const AppendArgs& a, bool aligned, cudaStream_t stream) {
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
  p.interleaved = a.interleaved;
  constexpr int kPer = ITER * 32 / (D / 8);
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
  return aligned ? cudaLaunchKernelEx(&cfg, paged_append_kernel<E, D, ITER, true>, p)
                 : cudaLaunchKernelEx(&cfg, paged_append_kernel<E, D, ITER, false>, p);
}

template <typename E, int D>
cudaError_t launch_iter(const PagedPool& pool, const AppendArgs& a, int num_sms, bool aligned,
                        cudaStream_t stream) {
  // Four heads a lane group once that still fills the GPU's warps; below it
  // one, so that a few tokens spread over the SMs.
  const int64_t groups = static_cast<int64_t>(a.T) * (a.hq + 2 * pool.n_kv_heads) * (D / 8) / 32;
  if (groups >= 4 * 64 * static_cast<int64_t>(num_sms)) return launch<E, D, 4>(pool, a, aligned, stream);
  return launch<E, D, 1>(pool, a, aligned, stream);
}

}  // namespace

cudaError_t launch_paged_append(const PagedPool& pool, const AppendArgs& a, int num_sms,
                                cudaStream_t stream) {
  const bool aligned = a.interleaved || a.rot % 16 == 0;
  if (pool.bf16)
    return pool.D == 128 ? launch_iter<__nv_bfloat16, 128>(pool, a, num_sms, aligned, stream)
                         : launch_iter<__nv_bfloat16, 64>(pool, a, num_sms, aligned, stream);
  return pool.D == 128 ? launch_iter<__half, 128>(pool, a, num_sms, aligned, stream)
                       : launch_iter<__half, 64>(pool, a, num_sms, aligned, stream);
}

}  // namespace dqg

DQG_STATUS_READER(read_status_append)
