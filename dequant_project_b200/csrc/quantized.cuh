// Device-side pieces shared by the kernels over a cache held in 8 bits: codes,
// and the search for the sequence that a unit of work belongs to.
#pragma once

#include "paged.cuh"
#include "quantized.h"

namespace dqg {

// Codes of eight bits. A block's scale is its largest magnitude over kMost.
struct Int8 {
  static constexpr float kMost = 127.f;
  // Four values (divided by the scale) to four codes.
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    const uint32_t ab = prmt(__float2int_rn(a), __float2int_rn(b), 0x0040);
    const uint32_t cd = prmt(__float2int_rn(c), __float2int_rn(d), 0x0040);
    return prmt(ab, cd, 0x5410);
  }
  // Four codes to four values: bytes plus 128 in the last bits of 2^23. (The
  // conversion instruction runs at an eighth of this rate.)
  static __device__ __forceinline__ void unpack4(uint32_t w, float* f) {
    w ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(prmt(w, 0x4b000000u, 0x7440 + i)) - 8388736.f;
  }
};
struct E4m3 {
  static constexpr float kMost = 448.f;
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    uint32_t w;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(w)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return w;
  }
  // Two codes (the low half of w) as two fp16 values, exactly.
  static __device__ __forceinline__ uint32_t half2(uint32_t w) {
    uint32_t h;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "mov.b32 {lo, hi}, %1;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
        : "=r"(h)
        : "r"(w));
    return h;
  }
  static __device__ __forceinline__ void unpack4(uint32_t w, float* f) {
    const float2 a = Elem<__half>::unpack(half2(w)), b = Elem<__half>::unpack(half2(w >> 16));
    f[0] = a.x;
    f[1] = a.y;
    f[2] = b.x;
    f[3] = b.y;
  }
};

// Finds the sequence that unit u belongs to when sequence b has count(b) of
// them, one sequence after the other: b, or -1 where there are fewer; *in: the
// unit's place in it. Taken by the whole block (`scratch`: 33 words of shared
// memory), which scans as many sequences at a time as it has threads.
template <class Count>
__device__ __forceinline__ int find_unit(int B, int64_t u, Count count, uint32_t* scratch, int64_t* in) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int b0 = 0; b0 < B; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    const uint32_t c = b < B ? count(b) : 0;
    uint32_t sum = c;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += t;
    }
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    int64_t before = 0;
    int found = -1;
    for (int w = 0; w < warps; ++w) {
      if (u < before + scratch[w]) {
        found = w;
        break;
      }
      before += scratch[w];
    }
    if (found >= 0) {
      if (warp == found) {
        const unsigned past = __ballot_sync(0xffffffffu, before + sum > u);
        const int l = __ffs(past) - 1;
        const uint32_t start = __shfl_sync(0xffffffffu, sum - c, l);
        __syncwarp();
        if (lane == 0) {
          scratch[warps] = b0 + 32 * warp + l;
          scratch[warps + 1] = static_cast<uint32_t>(u - before - start);
        }
      }
      __syncthreads();
      *in = scratch[warps + 1];
      return static_cast<int>(scratch[warps]);
    }
    u -= before;
    __syncthreads();
  }
  return -1;
}

}  // namespace dqg
