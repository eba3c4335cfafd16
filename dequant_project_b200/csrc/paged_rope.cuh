// One lane's part of a head's norm and rotation, shared by the kernels that
// store a batch of tokens (paged_append.cu, quantized_append.cu):
//
//   y     = x * rsqrt(mean(x^2) + eps) * w           (with a norm; per head)
//   (a,b) = (y_i, y_j),  j = i + R/2  or  (i, j) = (2p, 2p + 1)
//   a'    = a cos - b sin,  b' = b cos + a sin       (first R values; the rest pass)
//
// in fp32. A group of D / 16 lanes holds a head, and a lane two runs of eight
// values: in the half layout those at i and i + R/2, so that both values of a
// rotated pair lie in one lane and share a table entry; interleaved pairs lie
// in one lane anyway.
#pragma once

#include "paged.cuh"

namespace dqg {

enum RopeLayout {
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

template <typename E, int D, int LAYOUT>
struct RopeLane {
  static constexpr int kLanes = D / 16;  // lanes a head
  // Table entries of the lane's eight pairs (uneven: of its sixteen values).
  static constexpr int kTab = LAYOUT == kUneven ? 16 : 8;
  int c, rot, half, ea, eb;  // first values of the two runs
  bool pairs;
  float cs[kTab], sn[kTab];

  // Half layout: the first R / 16 lanes hold the pairs, the others what passes.
  __device__ __forceinline__ RopeLane(int c_, int rot_) : c(c_), rot(rot_), half(rot_ / 2) {
    pairs = LAYOUT != kHalf || c < rot / 16;
    ea = LAYOUT == kHalf ? (pairs ? 8 * c : 16 * c) : 16 * c;
    eb = LAYOUT == kHalf && pairs ? ea + rot / 2 : ea + 8;
  }
  // Rows of the tables: cos and sin of the token's position.
  __device__ __forceinline__ void entries(const float* cr, const float* sr) {
#pragma unroll
    for (int e = 0; e < kTab; ++e) {
      const int i = LAYOUT == kUneven ? (ea + e < half ? ea + e : ea + e - half) : 8 * c + e;
      const bool in = LAYOUT == kUneven ? ea + e < rot : i < half;
      cs[e] = in ? __ldg(cr + i) : 1.f;
      sn[e] = in ? __ldg(sr + i) : 0.f;
    }
  }
  // Norm (weights nw, or null) of the head whose runs are a and b; 1 / rms is
  // returned for rotate(). Taken by whole warps.
  __device__ __forceinline__ float norm(float* a, float* b, const E* nw, float eps) const {
    float r = 1.f;
    if (nw) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(a[e], a[e], fmaf(b[e], b[e], ss));
#pragma unroll
      for (int off = kLanes / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      r = rsqrtf(fmaf(ss, 1.f / D, eps));
      float wa[8], wb[8];
      unpack8<E>(__ldg(reinterpret_cast<const uint4*>(nw + ea)), wa);
      unpack8<E>(__ldg(reinterpret_cast<const uint4*>(nw + eb)), wb);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a[e] *= r * wa[e];
        b[e] *= r * wb[e];
      }
    }
    return r;
  }
  // head: where the head's values lie in memory (uneven layout).
  __device__ __forceinline__ void rotate(float* a, float* b, const E* head, const E* nw, float r) const {
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
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = ea + e, j = i < half ? i + half : i - half;
        float* t = e < 8 ? a + e : b + e - 8;
        if (i < rot) {
          float y = Elem<E>::load(head + j);
          if (nw) y *= r * Elem<E>::load(nw + j);
          *t = fmaf(*t, cs[e % kTab], i < half ? -(y * sn[e % kTab]) : y * sn[e % kTab]);
        }
      }
    }
  }
};

}  // namespace dqg
