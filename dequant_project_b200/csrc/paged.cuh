// Device-side pieces shared by the paged-cache kernels: 16-bit element types,
// tensor-map loads of page rows, and reads of a sequence's length.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.h"

namespace dqg {

template <typename E>
struct Elem;
template <>
struct Elem<__half> {
  static constexpr uint32_t kFormat = 0;  // tensor-core operand format
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  // a b + c, two values at a time.
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) { return hfma2_u32(a, b, c); }
  // All ones in each half that holds an infinity or a NaN.
  static __device__ __forceinline__ uint32_t non_finite(uint32_t v) { return __vcmpeq2(v & 0x7c007c00u, 0x7c007c00u); }
  // d += a b for one 16x16 by 16x8 tile (fp32 accumulators).
  static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr uint32_t kFormat = 1;
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) {
    return __bfloat162float(*p);
  }
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
  static __device__ __forceinline__ uint32_t non_finite(uint32_t v) { return __vcmpeq2(v & 0x7f807f80u, 0x7f807f80u); }
  static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// 2^x by the hardware's approximation (relative error about 2^-22; 2^-inf = 0).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One box of a 4-dimensional tensor map (this GPU's own memory) into shared
// memory. Coordinates out of range read zeros: a page index that no pool page
// has is the way to ask for a box of zeros.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar,
                                            int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// Order this thread's ordinary shared-memory accesses before later accesses of
// the asynchronous copy and tensor-core units to the same memory.
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// a / b of non-negative values; short where both fit 32 bits, as they mostly do.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}
// `total` units of work in shares of `each`, the last one shorter; at most n.
struct Shares {
  long long total, each;
  __device__ __forceinline__ void set(long long units, int n, int least) {
    total = units;
    each = quotient(units + n - 1, n);
    if (each < least) each = least;
  }
  __device__ __forceinline__ long long begin(int c) const {
    const long long b = c * each;
    return b < total ? b : total;
  }
  __device__ __forceinline__ int holder(long long unit) const {  // the share that holds a unit
    return static_cast<int>(quotient(unit, each));
  }
};

// A sequence's length, held to what its row of the table can address.
__device__ __forceinline__ int clamped_len(const int32_t* lens, int b, int limit) {
  const int n = __ldg(lens + b);
  return n < 0 ? 0 : (n > limit ? limit : n);
}

}  // namespace dqg
