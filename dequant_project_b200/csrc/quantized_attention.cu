// Decode attention over a cache held in 8 bits: one query token per sequence,
// lengths on the device, grouped KV heads. No reference counterpart (the
// reference models the cache's bytes, dequant/byte_model.py:214-219).
//
//   o[b, h] = sum_t p_t s_v(t) code_v(t) / sum_t p_t,
//   p_t = exp(scale s_k(t) q[b, h] . code_k(t) - m)
//
// over the complete blocks of sequence b and then the 16-bit rows of its open
// block (s = 1); zero where there is none.
//
// The work is cut as in paged_attention.cu (paged_decode.cuh): equal shares of
// tiles of 112 positions, pieces of cut items joined in order by a second
// kernel. One warp copies a tile's code rows by tensor-map boxes of 16 and its
// scales by cp.async into a ring; seven warps take 16 positions each, which
// lie in one block, so that a warp's scales are two numbers (eight warps in
// all, two CTAs per SM: 128 registers a thread). Positions are the
// m side of mma.m16n8k16 and query heads its n side (8 of them, or 16 in two
// products): S = K Q^T, then O^T += V^T P, with the weights transposed between
// by movmatrix. With heads on the m side, as in the 16-bit kernel, half or more
// of the products' rows and of the accumulators would be empty for the usual
// one to eight heads a KV head.
//
// Codes are read from shared memory sixteen bytes a lane and become operands in
// registers, exactly (Pairs), in whatever order of the summed index that gives,
// the queries' being the same. Beside e4m3 codes bf16 queries become fp16 times
// a power of two for each head, the largest between 2^14 and 2^15: what that
// loses is below 2^-39 of the largest; beside int8 codes they are digits (Pairs).
// Scores are scaled in fp32. So are the weights: besides the softmax's reference
// (of the scores) the sum over values has one of its own, of the score plus log2
// s_v, so that a 16-bit weight is relative to the largest p s_v met, whatever the
// blocks' scales are. Both references move, and the sums are rescaled, only when a
// slice exceeds one by more than 2^kMaxGrowth; of fp16's range (2^-24 to 2^16) a
// weight loses below 2^-32 of the largest. (A weight's one rounding to fp16 adds up
// to a tenth to the output's own error: 2.2e-4 instead of 2.1e-4 for 2049 positions
// in fp16.) Open rows go through products of their own type, with weights relative
// to their own largest. The warps' parts, and the pieces of cut items, are merged as
// means of the values, so that what is finite in the cache gives a finite result.
//
// HBM bounds the large calls: 64 sequences of 0 to 16000 positions (64 and 8
// heads of 128, int8, 0.63 GB) take 117 to 119 us, joining included, 5.3 TB/s (122
// to 129 in a longer stream, where the power cap lowers the clock); 64 of 8000 (1
// GB) 180 us, 5.8 TB/s, and e4m3 171 us, 6.1 TB/s (200 and 188 in a stream of 0.4
// s). What is left between is items' starts and ends and the second kernel. Short
// calls are latency: one sequence of 2049 positions of 32 heads 11.5 us for 2.6 us of
// bytes. Steps that counted, 64 sequences: a warp a position on plain lanes 4154 us;
// tensor products 147; seven consumer warps at 128 registers, two CTAs, 136; integer
// products of the keys and the merge in rounds of four heads 119; a third digit of
// the queries 2 % more; no code for a prefix 1 % less (2049 positions 12.5 -> 11.5).
//
// Waits are bounded, as in paged_attention.cu: a consumer warp whose wait ran
// out goes on without data and makes its results NaN.
#include <cstdint>

#include "paged_decode.cuh"
#include "quantized.cuh"

namespace dqg {
namespace {

constexpr int kWarps = 7;              // consumer warps, 16 positions each
constexpr int kTile = 16 * kWarps;     // positions per tile
constexpr int kOpen = 48;              // open rows per tile: their keys fit the codes' place
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kQuerySlots = 4;         // items whose queries are held at most
constexpr int kMergeRows = 4;          // query heads per round of the warps' merge
constexpr float kMaxGrowth = 8.f, kHeadroom = 7.f;  // log2 units
constexpr float kOpenTop = 14.f;  // of fp16 open rows' weights, the largest

struct Params : DecodeParams {
  static constexpr bool kPrefix = false;
  const float* k_scale;
  const float* v_scale;
  const void* k_open;
  const void* v_open;
  const int32_t* open_slots;
  int64_t scale_page_stride, scale_head_stride, open_stride, open_head_stride, n_open;
  int block_shift;
};

// Tiles of complete blocks, and of the open block's rows.
__device__ __forceinline__ int tiles_of(const Params& p, int len) {
  const int open = len & ((1 << p.block_shift) - 1);
  return max(1, (len - open + kTile - 1) / kTile + (open + kOpen - 1) / kOpen);
}

template <int kOff = 0>
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr), "n"(kOff));
  return v;
}
template <int kOff = 0>
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2 + %3];" : "=r"(v.x), "=r"(v.y) : "r"(addr), "n"(kOff));
  return v;
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
  return m;
}
__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// Arrives once this thread's earlier cp.async copies are complete.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Codes as operands. Values, four codes a word, become two pairs of fp16
// numbers: bytes (0, 2) and (1, 3) where kStride is 2, (0, 1) and (2, 3) where
// it is 1. e4m3: one conversion for two. int8: the byte with its sign bit turned
// over, as the fraction of a subnormal number, (code + 128) / 2^24: one or two
// integer instructions a pair; the bias goes out of the sums again (a product
// more per slice sums 128 p). Bytes put into the fraction of 1024 and made small
// again by an addition took 64 more instructions of about 430 a slice.
// Keys: e4m3 the same way. int8 codes enter integer products as they are, beside
// the queries as integers of 23 bits, relative to their head's largest, in three int8
// digits: what that loses is at most 2^-23 of the largest, so that a channel far above
// the others takes nothing that matters from them. (Two digits, 2^-16, took 1 to 2 %
// less time, and a channel of 4000 made outputs 0.04 of a value off. Codes as fp16
// numbers, as the values, beside the queries' own took 9 % more: 64 sequences of 8000
// 195 us instead of 180 in a graph.)
template <class Code>
struct Pairs;
template <>
struct Pairs<Int8> {
  static constexpr int kStride = 2, kUnit = 24;
  static constexpr bool kInteger = true;
  static constexpr uint32_t kBias = 0x00800080u;  // 128 / 2^24, twice
  static __device__ __forceinline__ void expand(uint32_t w, uint32_t& a, uint32_t& b) {
    a = (w & 0x00ff00ffu) ^ kBias;
    b = ((w >> 8) & 0x00ff00ffu) ^ kBias;
  }
};
template <>
struct Pairs<E4m3> {
  static constexpr int kStride = 1, kUnit = 0;
  static constexpr bool kInteger = false;
  static constexpr uint32_t kBias = 0;
  static __device__ __forceinline__ void expand(uint32_t w, uint32_t& a, uint32_t& b) {
    a = E4m3::half2(w);
    b = E4m3::half2(w >> 16);
  }
};
// d += a b of int8 values, one 16x32 by 32x8 tile. Sums below 2^22 that begin at
// kIntZero are the bits of that float plus the sum.
__device__ __forceinline__ void mma_s8(int* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr int kIntZero = 0x4b400000;  // 1.5 * 2^23
constexpr float kDigitMost = 4161407.f;  // 63, 127, 127 in digits of eight bits
__device__ __forceinline__ float int_sum(int bits) { return __int_as_float(bits) - 12582912.f; }

// Row of a tile that row n of a product takes: conflict-free reads of sixteen
// bytes a lane by eight rows of four lanes (keys) as by four of eight (values).
__device__ __forceinline__ int row_of(int n) { return n ^ ((n & 1) << 2); }

// Byte offset of 16-byte chunk `chunk` of code row `row`, swizzled as the
// tensor map writes it (128 bytes for rows of 128, 64 for rows of 64).
template <int D>
__device__ __forceinline__ uint32_t code_off(int row, int chunk) {
  return D == 128 ? row * 128 + ((chunk ^ (row & 7)) << 4) : row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}

template <int D, int NB>
struct Layout {
  static constexpr int kCtasPerSm = NB == 1 ? 2 : 1;
  static constexpr int kStages = NB == 1 ? 3 : 6;
  static constexpr int kTileBytes = kTile * D;
  static_assert(kOpen * D * 2 <= kTileBytes, "open rows");
  static constexpr int kRing = kStages * 2 * kTileBytes;
  static constexpr int kQuery = 16 * D * 2;
  static constexpr int kMerge = kWarps * kMergeRows * D * 4;
  static constexpr int kStats = 3 * kWarps * 16 * 4;
  static constexpr int kScaleBytes = kStages * 2 * kWarps * 4;
  static constexpr int kSmem =
      1024 + kRing + kQuery + kMerge + kStats + kScaleBytes + 2 * (kStages + kQuerySlots) * 8 + static_cast<int>(sizeof(Share));
};

template <typename E, class Code, int D, int NB>
__global__ void __launch_bounds__(kThreads, Layout<D, NB>::kCtasPerSm)
    quantized_decode_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap kmap,
                            const __grid_constant__ CUtensorMap vmap) {
  using L = Layout<D, NB>;
  constexpr int kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  // Queries of the items ahead; reads of 8 or 16 rows run past a short slot, at
  // worst into the merge buffer (columns whose results nobody takes).
  uint8_t* qs = smem + L::kRing;
  float* os = reinterpret_cast<float*>(qs + L::kQuery);          // [warp][kMergeRows][D]
  float* ms = os + L::kMerge / 4;                                // [warp][16]: the scores' reference,
  float* vs = ms + kWarps * 16;                                  // the values',
  float* ls = vs + kWarps * 16;                                  // and the sum
  float* scales = ls + kWarps * 16;                              // [stage][slice][key, value]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + L::kScaleBytes / 4);
  uint64_t* empty = full + kStages;
  uint64_t* q_full = empty + kStages;
  uint64_t* q_empty = q_full + kQuerySlots;
  Share* share = reinterpret_cast<Share*>(q_empty + kQuerySlots);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + i, 1 + 2 * kWarps);
      mbar_init(empty + i, kWarps);
    }
    for (int i = 0; i < kQuerySlots; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, kWarps);
    }
    fence_mbar_init();
    tma_prefetch_map(&kmap);
    tma_prefetch_map(&vmap);
  }
  pdl_wait_prior_grid();
  if (warp == 0) {
    const Share s = find_share(p, blockIdx.x, gridDim.x);
    if (lane == 0) *share = s;
  }
  __syncthreads();
  pdl_launch_dependents();
  Share s = *share;
  const int q_rows = min(16, p.g), q_slots = min(kQuerySlots, 16 / q_rows);
  const int block = 1 << p.block_shift;

  if (warp == kWarps) {
    // ---- the copying warp.
    const uint64_t policy = policy_evict_last();
    int it = 0, item = 0;
    bool ok = !(p.starved >> kWarps & 1);
    while (s.count > 0 && ok) {
      const Item i = item_of(p, s);
      if (i.x1 == i.x0) {  // the cut falls before its first tile
        advance(p, s, i.units);
        continue;
      }
      const int done = i.len & ~(block - 1), whole = (done + kTile - 1) / kTile;
      if (lane == 0 && __ldg(p.lens + s.b) != i.len) atomicOr(&g_status, kStatusBadIndex);
      const int qi = item % q_slots;
      if (item >= q_slots && !warp_wait(q_empty + qi, ((item / q_slots) & 1) ^ 1, p.wait_ns)) break;
      if (lane == 0) mbar_arrive_expect_tx(q_full + qi, i.rows * D * 2);
      __syncwarp();
      if (lane < i.rows)
        bulk_g2s(qs + (qi * q_rows + lane) * D * 2, static_cast<const E*>(p.q) + s.b * p.q_stride_seq +
                 (i.head0 + lane) * p.q_stride_head, D * 2, q_full + qi, policy);
      ++item;
      // A lane a slice of 16 positions, of keys and then of values: its box and
      // its block's scale. Pages are read from the table one tile ahead: their
      // latency would be a tile's time.
      const int slice = lane % kWarps, n_pages = static_cast<int>(p.n_pages);
      const bool values = lane >= kWarps;
      auto page_of = [&](int x) {
        const int t = x * kTile + slice * 16;
        return lane < 2 * kWarps && t < done ? __ldg(i.table + (t >> p.page_shift)) : 0;
      };
      int page = page_of(i.x0), next = 0;
      for (int x = i.x0; x < i.x1; ++x, ++it, page = next) {
        const int st = it % kStages;
        uint8_t* dst = smem + st * 2 * L::kTileBytes;
        if (x + 1 < i.x1) next = page_of(x + 1);
        if (x < whole || i.len == done) {
          if (it >= kStages && !warp_wait(empty + st, ((it / kStages) & 1) ^ 1, p.wait_ns)) {
            ok = false;
            break;
          }
          // No position, or no such page: zeros.
          const bool some = x * kTile + slice * 16 < done, good = some && page >= 0 && page < n_pages;
          if (some && !good) atomicOr(&g_status, kStatusBadIndex);
          if (lane == 0) mbar_arrive_expect_tx(full + st, 2 * L::kTileBytes);
          __syncwarp();
          if (lane < 2 * kWarps) {
            const int in_page = (x * kTile + slice * 16) & ((1 << p.page_shift) - 1);
            tma_load_4d(smem_u32(dst) + lane * (16 * D), values ? &vmap : &kmap, full + st, 0, in_page, i.kvh,
                        good ? page : n_pages);
            float* to = scales + (st * kWarps + slice) * 2 + (values ? 1 : 0);
            if (good) {
              cp_async4(smem_u32(to), (values ? p.v_scale : p.k_scale) + page * p.scale_page_stride +
                        i.kvh * p.scale_head_stride + (in_page >> p.block_shift));
              cp_async_arrive(full + st);
            } else {
              *to = 0.f;
              mbar_arrive(full + st);  // (releases the store; the other form waits for copies only)
            }
          }
        } else {
          // The open rows, as they are.
          const int first = (x - whole) * kOpen, rows = min(kOpen, i.len - done - first);
          const int64_t slot = __ldg(p.open_slots + s.b);
          const bool good = slot >= 0 && slot < p.n_open;
          if (it >= kStages && !warp_wait(empty + st, ((it / kStages) & 1) ^ 1, p.wait_ns)) {
            ok = false;
            break;
          }
          if (!good) {
            for (int c = lane; c < 2 * L::kTileBytes / 16; c += 32) reinterpret_cast<uint4*>(dst)[c] = make_uint4(0, 0, 0, 0);
            if (lane == 0) atomicOr(&g_status, kStatusBadIndex);
            __syncwarp();
            fence_async_shared();  // before the ring's next copy to this place
          }
          if (lane == 0) {
            mbar_arrive_expect_tx(full + st, good ? 2 * rows * D * 2 : 0);
            if (good) {
              const int64_t at = slot * p.open_stride + i.kvh * p.open_head_stride + first * D;
              bulk_g2s(dst, static_cast<const E*>(p.k_open) + at, rows * D * 2, full + st, policy);
              bulk_g2s(dst + L::kTileBytes, static_cast<const E*>(p.v_open) + at, rows * D * 2, full + st, policy);
            }
          }
          __syncwarp();
          if (lane < 2 * kWarps) mbar_arrive(full + st);
        }
      }
      advance(p, s, i.units);
    }
    // Copies still in flight land before the CTA's memory goes (bounded).
    for (int i = item < q_slots ? 0 : item - q_slots; i < item; ++i)
      if (!warp_wait(q_full + i % q_slots, (i / q_slots) & 1, p.wait_ns)) break;
    for (int i = it < kStages ? 0 : it - kStages; i < it; ++i)
      if (!warp_wait(full + i % kStages, (i / kStages) & 1, p.wait_ns)) break;
  } else {
    using Pair = Pairs<Code>;
    constexpr int kSums = D / 16 + (Pair::kInteger ? 1 : 0);  // products a slice; the last one sums the bias
    constexpr int kDigits = Pair::kInteger ? 3 : 2;  // words of queries a product takes
    const int gid = lane >> 2, c = lane & 3;
    const uint32_t ring = smem_u32(smem);
    const int p0 = warp * 16;
    // Where this lane reads in a stage's keys and values; rows 8 further lie
    // 8 rows' bytes behind.
    uint32_t k_at[D / 64], v_at[2];
#pragma unroll
    for (int h = 0; h < D / 64; ++h) k_at[h] = ring + code_off<D>(p0 + row_of(gid), c + 4 * h);
#pragma unroll
    for (int r = 0; r < 2; ++r)
      v_at[r] = ring + L::kTileBytes + (D == 128 ? code_off<D>(p0 + row_of(2 * c + r), gid)
                                                 : code_off<D>(p0 + row_of(2 * c + r), gid >> 1) + (gid & 1) * 8);
    int stage = 0, item = 0;
    uint32_t parity = 0;
    // Once a wait has run out no later one is taken.
    bool ok = !(p.starved >> warp & 1), cut_first = false;
    auto await = [&](uint64_t* bar, uint32_t phase) { return ok = ok && warp_wait(bar, phase, p.wait_ns); };
    while (s.count > 0) {
      const Item i = item_of(p, s);
      if (i.x1 == i.x0) {
        advance(p, s, i.units);
        continue;
      }
      const int done = i.len & ~(block - 1), whole = (done + kTile - 1) / kTile;
      const int qi = item % q_slots;
      await(q_full + qi, (item / q_slots) & 1);
      // Queries as B fragments: columns are heads; a lane holds the values at
      // 64 h + 16 c to + 15, four a product (fp16) or eight (digits).
      uint32_t qf[NB][D / 16][kDigits];  // digits: [word][high, middle, low]
      float unit[NB][2];           // what scores of heads 2 c and 2 c + 1 are multiplied by, but for the block's scale
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const uint32_t row = smem_u32(qs) + (qi * q_rows + nb * 8 + gid) * (D * 2) + c * 32;
        uint32_t w[D / 8];
        uint32_t most = 0;
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
          const uint4 v = lds128(row + (h >> 1) * 128 + (h & 1) * 16);
          w[4 * h] = v.x;
          w[4 * h + 1] = v.y;
          w[4 * h + 2] = v.z;
          w[4 * h + 3] = v.w;
        }
#pragma unroll
        for (int h = 0; h < D / 8; ++h) most = __vmaxu2(most, w[h] & 0x7fff7fffu);
        most = max(most & 0xffffu, most >> 16);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        float f = p.scale_log2;
        if constexpr (Pair::kInteger) {
          // Digits by a sum with 1.5 * 2^23, whose last bits are the integer, and with
          // 128 in each digit's place, which makes all three positive bytes. (A
          // largest value that is not finite makes the head's unit so.)
          const float largest = Elem<E>::unpack(most).x, up = fminf(kDigitMost / largest, 1e38f);
          f *= up < 1e38f ? largest / kDigitMost : (largest == largest ? 1e-38f : NAN);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const float2 x = Elem<E>::unpack(w[2 * k]), y = Elem<E>::unpack(w[2 * k + 1]);
            const float v[4] = {x.x, x.y, y.x, y.y};
            uint32_t n[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) n[e] = __float_as_uint(fmaf(v[e], up, 12582912.f)) + (0x808080u - kIntZero);
            const uint32_t a = prmt(n[0], n[1], 0x5140), b = prmt(n[2], n[3], 0x5140);
            qf[nb][k][0] = prmt(prmt(n[0], n[1], 0x0062), prmt(n[2], n[3], 0x0062), 0x5410) ^ 0x80808080u;
            qf[nb][k][1] = prmt(a, b, 0x7632) ^ 0x80808080u;
            qf[nb][k][kDigits - 1] = prmt(a, b, 0x5410) ^ 0x80808080u;
          }
        } else {
          if (Elem<E>::kFormat == 1) {
            // bf16 to fp16, times a power of two for the head.
            const int e = min(max(static_cast<int>(most >> 7), 15), 254);  // exponent of the largest, biased
            const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 + 127 - e) << 23);  // 2^(14 - (e - 127))
#pragma unroll
            for (int h = 0; h < D / 8; ++h) {
              const float2 x = Elem<E>::unpack(w[h]);
              w[h] = Elem<__half>::pack(x.x * up, x.y * up);
            }
            f *= __uint_as_float(static_cast<uint32_t>(e - 14) << 23);  // 2^((e - 127) - 14)
          }
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            qf[nb][k][0] = w[2 * k];
            qf[nb][k][1] = w[2 * k + 1];
          }
        }
        unit[nb][0] = __shfl_sync(0xffffffffu, f, 8 * c);  // of lanes with gid = 2 c
        unit[nb][1] = __shfl_sync(0xffffffffu, f, 8 * c + 4);
      }
      float o[NB][kSums][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int k = 0; k < kSums; ++k) o[nb][k][0] = o[nb][k][1] = o[nb][k][2] = o[nb][k][3] = 0.f;
      // References of heads 2 c and 2 c + 1, kHeadroom below a maximum that the
      // true one exceeds by kMaxGrowth at most, of the scores and of what the
      // values are weighed with; l: this lane's part of the sum.
      float ref[NB][2], ref_v[NB][2], l[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          ref[nb][e] = ref_v[nb][e] = -3.4e38f;
          l[nb][e] = 0.f;
        }
      // Weights of a slice, whose scores are sc * f (log2 units; entries 2 r + e:
      // row gid + 8 r, head 2 c + e): for the softmax's sum into l, and for the
      // values, whose scale is 2^lv, in place of sc.
      auto weigh = [&](float (&sc)[NB][4], const float (&f)[NB][2], float lv) {
        float a[NB][4], b[NB][4], most = -INFINITY;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[nb][e] = fmaf(sc[nb][e], f[nb][e & 1], -ref[nb][e & 1]);
            b[nb][e] = fmaf(sc[nb][e], f[nb][e & 1], lv - ref_v[nb][e & 1]);
            most = max3(most, a[nb][e], b[nb][e]);
          }
        if (__any_sync(0xffffffffu, most > kHeadroom + kMaxGrowth)) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(sc[nb][e] * f[nb][e], sc[nb][e + 2] * f[nb][e]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16)) - kHeadroom;
              // (Each column by itself: those of no head hold anything.)
              if (mx - ref[nb][e] > kMaxGrowth) {
                l[nb][e] *= exp2_approx(ref[nb][e] - mx);
                ref[nb][e] = mx;
              }
              if (mx + lv - ref_v[nb][e] > kMaxGrowth) {
                const float g = exp2_approx(ref_v[nb][e] - (mx + lv));
                ref_v[nb][e] = mx + lv;
#pragma unroll
                for (int k = 0; k < kSums; ++k) {
                  o[nb][k][e] *= g;
                  o[nb][k][e + 2] *= g;
                }
              }
#pragma unroll
              for (int r = 0; r < 4; r += 2) {
                a[nb][e + r] = fmaf(sc[nb][e + r], f[nb][e], -ref[nb][e]);
                b[nb][e + r] = fmaf(sc[nb][e + r], f[nb][e], lv - ref_v[nb][e]);
              }
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            l[nb][e & 1] += exp2_approx(a[nb][e]);
            sc[nb][e] = exp2_approx(b[nb][e]);
          }
      };
      for (int x = i.x0; x < i.x1; ++x) {
        const uint32_t at = stage * 2 * L::kTileBytes;
        if (await(full + stage, parity)) {
          if (x < whole || i.len == done) {
            if (x * kTile + p0 < done) {
              const float2 both = *reinterpret_cast<const float2*>(scales + (stage * kWarps + warp) * 2);
              const float ks = both.x, lv = log2_approx(both.y) + Pair::kUnit;
              float sc[NB][4], f[NB][2];
              int sums[NB][3][4];
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                f[nb][0] = unit[nb][0] * ks;
                f[nb][1] = unit[nb][1] * ks;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  sc[nb][e] = 0.f;
                  sums[nb][0][e] = kIntZero;
                  sums[nb][1][e] = sums[nb][2][e] = 0;
                }
              }
#pragma unroll
              for (int h = 0; h < D / 64; ++h) {
                const uint4 a = lds128(k_at[h] + at), b = lds128<8 * D>(k_at[h] + at);
                const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
                if constexpr (Pair::kInteger) {
#pragma unroll
                  for (int k = 0; k < 4; k += 2)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                      for (int e = 0; e < kDigits; ++e)
                        mma_s8(sums[nb][e], aw[k], bw[k], aw[k + 1], bw[k + 1], qf[nb][4 * h + k][e],
                               qf[nb][4 * h + k + 1][e]);
                } else {
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    uint32_t w[4];
                    Pair::expand(aw[k], w[0], w[2]);
                    Pair::expand(bw[k], w[1], w[3]);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                      Elem<__half>::mma(sc[nb], w, qf[nb][4 * h + k][0], qf[nb][4 * h + k][1]);
                  }
                }
              }
              if constexpr (Pair::kInteger) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    sc[nb][e] = fmaf(int_sum(sums[nb][0][e]), 65536.f, __int2float_rn(sums[nb][1][e] * 256 + sums[nb][2][e]));
              }
              // A lane's D / 8 values of four rows: a word of each gives two
              // products' halves.
              constexpr uint32_t kLow = Pair::kStride == 2 ? 0x5410 : 0x5140;
              constexpr uint32_t kHigh = Pair::kStride == 2 ? 0x7632 : 0x7362;
              uint32_t vw[4][D / 32];
              auto load_values = [&] {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const uint32_t from = v_at[r & 1] + at;
                  if (D == 128) {
                    const uint4 v = r & 2 ? lds128<8 * D>(from) : lds128(from);
                    vw[r][0] = v.x;
                    vw[r][1] = v.y;
                    vw[r][2 % (D / 32)] = v.z;
                    vw[r][3 % (D / 32)] = v.w;
                  } else {
                    const uint2 v = r & 2 ? lds64<8 * D>(from) : lds64(from);
                    vw[r][0] = v.x;
                    vw[r][1] = v.y;
                  }
                }
              };
              // (Ahead of the weights where there are registers for it: with three
              // digits of queries and 128 registers 64 sequences took 2 % longer.)
              constexpr bool kLate = Pair::kInteger && NB == 1;
              if (!kLate) load_values();
              weigh(sc, f, lv);
              if (kLate) load_values();
              uint32_t pf[NB][2];
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                pf[nb][0] = transposed(Elem<__half>::pack(sc[nb][0], sc[nb][1]));
                pf[nb][1] = transposed(Elem<__half>::pack(sc[nb][2], sc[nb][3]));
              }
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                const uint32_t sel = k & 1 ? kHigh : kLow;
                uint32_t w[4];
                Pair::expand(prmt(vw[0][k / 2], vw[1][k / 2], sel), w[0], w[1]);
                Pair::expand(prmt(vw[2][k / 2], vw[3][k / 2], sel), w[2], w[3]);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) Elem<__half>::mma(o[nb][k], w, pf[nb][0], pf[nb][1]);
              }
              if (Pair::kInteger) {
                const uint32_t ones[4] = {Pair::kBias, Pair::kBias, Pair::kBias, Pair::kBias};
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) Elem<__half>::mma(o[nb][kSums - 1], ones, pf[nb][0], pf[nb][1]);
              }
            }
          } else if (p0 < min(kOpen, i.len - done - (x - whole) * kOpen)) {
            // Open rows, in their own type: rows of the products are the tile's.
            const uint32_t kst = ring + at, vst = kst + L::kTileBytes;
            const int rows = i.len - done - (x - whole) * kOpen - p0;  // of this warp's 16, or more
            float sc[NB][4];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.f;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t off = (k / 4) * 128 + c * 32 + (k % 4) * 8;
              const uint2 a = lds64(kst + (p0 + gid) * (D * 2) + off), b = lds64(kst + (p0 + 8 + gid) * (D * 2) + off);
              const uint32_t w[4] = {a.x, b.x, a.y, b.y};
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                const uint2 q = lds64(smem_u32(qs) + (qi * q_rows + nb * 8 + gid) * (D * 2) + off);
                Elem<E>::mma(sc[nb], w, q.x, q.y);
              }
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[nb][e] = gid + 8 * (e >> 1) < rows ? sc[nb][e] : -INFINITY;
            // Their weights refer to their own largest, and the products are added to
            // the sums in fp32: relative to a block's weights, which have its scale in
            // them (and int8's 2^24), fp16 would not hold them beside values thousands
            // of times theirs. (The bias of int8 sums goes out first, so that it takes
            // no bits of what is added.)
            auto value_pair = [&](int k, int r) {
              // What lies behind the last row may be anything: a zero weight
              // times an infinity would not be zero.
              const int row = 2 * c + (r & 1) + (r & 2 ? 8 : 0);
              uint32_t w = 0;
              if (row < rows)
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(vst + (p0 + row) * (D * 2) + gid * (D / 4) + k * 4));
              return w;
            };
            float top = kOpenTop;
            if constexpr (Elem<E>::kFormat == 1) {
              // bf16: 2^64 over the largest value's power of two, so that sums of
              // values of any size are fp32 numbers (and weights normal ones).
              uint32_t most = 0;
#pragma unroll
              for (int k = 0; k < D / 16; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) most = __vmaxu2(most, value_pair(k, r) & 0x7fff7fffu);
#pragma unroll
              for (int off = 16; off >= 1; off >>= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, off));
              most = max(most & 0xffffu, most >> 16);
              top = static_cast<float>(min(64 + 127 - static_cast<int>(most >> 7), 120));
            }
            float g[NB][2], keep[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float mx = fmaxf(sc[nb][e], sc[nb][e + 2]) * p.scale_log2;
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = max3(mx, __shfl_xor_sync(0xffffffffu, mx, 16), -3.4e38f);
                if (mx - kHeadroom - ref[nb][e] > kMaxGrowth) {
                  l[nb][e] *= exp2_approx(ref[nb][e] - (mx - kHeadroom));
                  ref[nb][e] = mx - kHeadroom;
                }
                const float own = mx - top, to = fmaxf(ref_v[nb][e], own);
                keep[nb][e] = exp2_approx(ref_v[nb][e] - to);
                g[nb][e] = exp2_approx(own - to);
                ref_v[nb][e] = to;
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                  l[nb][e] += exp2_approx(fmaf(sc[nb][e + r], p.scale_log2, -ref[nb][e]));
                  sc[nb][e + r] = exp2_approx(fmaf(sc[nb][e + r], p.scale_log2, -own));
                }
              }
            }
            uint32_t pf[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              pf[nb][0] = transposed(Elem<E>::pack(sc[nb][0], sc[nb][1]));
              pf[nb][1] = transposed(Elem<E>::pack(sc[nb][2], sc[nb][3]));
            }
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t w[4] = {value_pair(k, 0), value_pair(k, 1), value_pair(k, 2), value_pair(k, 3)};
              const uint32_t v[4] = {prmt(w[0], w[1], 0x5410), prmt(w[0], w[1], 0x7632), prmt(w[2], w[3], 0x5410),
                                     prmt(w[2], w[3], 0x7632)};
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
                Elem<E>::mma(d, v, pf[nb][0], pf[nb][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float before = o[nb][k][e] - (Pair::kInteger ? o[nb][kSums - 1][e & 1] : 0.f);
                  o[nb][k][e] = fmaf(d[e], g[nb][e & 1], before * keep[nb][e & 1]);
                }
              }
            }
            if (Pair::kInteger) {
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) o[nb][kSums - 1][0] = o[nb][kSums - 1][1] = 0.f;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(empty + stage);
        }
        if (++stage == kStages) {
          stage = 0;
          parity ^= 1;
        }
      }
      if (Pair::kInteger) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nb][k][e] -= o[nb][kSums - 1][e & 1];
      }
      // The queries' place is free once their reads have come back, not once
      // they are issued: here every fragment is used.
      {
        uint32_t x = 0;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int k = 0; k < D / 16; ++k) for (int t = 0; t < kDigits; ++t) x ^= qf[nb][k][t];
        asm volatile("" ::"r"(x) : "memory");
      }
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(q_empty + qi);
      ++item;

      // The item's (or piece's) result: the warps' references and sums first,
      // then their parts, four heads a round.
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 4);
          l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 8);
          l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 16);
          if (gid == 0) {
            const int at = warp * 16 + nb * 8 + 2 * c + e;
            // (-inf: no position yet, as in the pieces.)
            ms[at] = ref[nb][e] == -3.4e38f ? -INFINITY : ref[nb][e];
            vs[at] = ref_v[nb][e] == -3.4e38f ? -INFINITY : ref_v[nb][e];
            ls[at] = ok ? l[nb][e] : NAN;
          }
        }
      named_sync(1, 32 * kWarps);
      const bool all = i.x0 == 0 && i.x1 == i.tiles;
      const int64_t row0 = (2 * static_cast<int64_t>(blockIdx.x) + (i.x0 > 0 ? 0 : 1)) * p.rows;
      if (threadIdx.x < i.rows) {
        // A head's maximum, its sum, what each warp's part is multiplied by, and
        // what their sum is, to be the mean of the values: the sum's reciprocal and
        // the power of two between the references, in two halves since all of it
        // may be no fp32 number (a scale is up to 2^121).
        const int row = threadIdx.x;
        float mx = -INFINITY, mv = -INFINITY, den = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          mx = fmaxf(mx, ms[w * 16 + row]);
          mv = fmaxf(mv, vs[w * 16 + row]);
        }
        const float mu = mx == -INFINITY ? 0.f : mx, nu = mv == -INFINITY ? mu : mv;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          den = fmaf(ls[w * 16 + row], exp2_approx(ms[w * 16 + row] - mu), den);
          vs[w * 16 + row] = exp2_approx(vs[w * 16 + row] - nu);
        }
        const float half = exp2_approx(0.5f * (nu - mu));
        ls[row] = den == 0.f ? 0.f : half * __frcp_rn(den);
        ms[row] = half;
        if (!all) {
          p.m[row0 + row] = mx;
          p.l[row0 + row] = den;
        }
      }
      if (i.x0 == 0 && !all) {
        cut_first = true;
        if (threadIdx.x == 0) {
          const int last = s.all.holder(s.pos - s.x + i.tiles + p.item_tiles - 1);
          p.desc[blockIdx.x] = Desc{s.b, s.hv, static_cast<int>(blockIdx.x), last - static_cast<int>(blockIdx.x) + 1};
        }
      }
#pragma unroll
      for (int r = 0; r < 2 * NB; ++r) {
        if (kMergeRows * r >= i.rows) break;
        if (c / 2 == r % 2) {
          // Sixteen (or eight) values of a head a lane; their chunks are
          // swizzled by gid against bank conflicts.
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int k = 0; k < D / 32; ++k)
              *reinterpret_cast<float4*>(os + (warp * kMergeRows + 2 * (c % 2) + e) * D + gid * (D / 8) +
                                         (k ^ ((gid >> 1) & (D / 32 - 1))) * 4) =
                  make_float4(o[r / 2][2 * k][e], o[r / 2][2 * k][e + 2], o[r / 2][2 * k + 1][e], o[r / 2][2 * k + 1][e + 2]);
        }
        named_sync(1, 32 * kWarps);
        for (int cell = threadIdx.x; cell < kMergeRows * (D / 4); cell += 32 * kWarps) {
          const int j = cell / (D / 4), d4 = cell % (D / 4), row = kMergeRows * r + j;
          if (row < i.rows) {
            const int g8 = d4 / (D / 32), at = g8 * (D / 8) + ((d4 ^ (g8 >> 1)) & (D / 32 - 1)) * 4;
            float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              const float f = vs[w * 16 + row];
              const float4 v = *reinterpret_cast<const float4*>(os + (w * kMergeRows + j) * D + at);
              num.x = fmaf(v.x, f, num.x);
              num.y = fmaf(v.y, f, num.y);
              num.z = fmaf(v.z, f, num.z);
              num.w = fmaf(v.w, f, num.w);
            }
            const float f = ls[row], half = ms[row];
            num = make_float4(num.x * f * half, num.y * f * half, num.z * f * half, num.w * f * half);
            if (all)
              store4<E, D>(p, s.b, i.head0 + row, d4, 1.f, num);
            else
              *reinterpret_cast<float4*>(p.part + (row0 + row) * D + d4 * 4) = num;
          }
        }
        named_sync(1, 32 * kWarps);
      }
      advance(p, s, i.units);
    }
    if (threadIdx.x == 0 && !cut_first) p.desc[blockIdx.x] = Desc{0, 0, 0, 0};
  }
}

template <typename E, class Code, int D, int NB>
cudaError_t launch(Params p, const CUtensorMap& kmap, const CUtensorMap& vmap, int num_sms, cudaStream_t stream) {
  using L = Layout<D, NB>;
  static int configured[64] = {0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(quantized_decode_kernel<E, Code, D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             L::kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = 1;
  }
  p.n_ctas = L::kCtasPerSm * num_sms;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.n_ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, quantized_decode_kernel<E, Code, D, NB>, p, kmap, vmap);
  if (e != cudaSuccess) return e;
  return launch_join<E, D, true>(p, cfg);
}

template <typename E, class Code>
cudaError_t launch_for(const Params& p, int D, const CUtensorMap& kmap, const CUtensorMap& vmap, int num_sms,
                       cudaStream_t stream) {
  // Heads of a KV head: one product's eight columns, or two's sixteen (and row
  // blocks of sixteen beyond).
  if (p.g <= 8)
    return D == 128 ? launch<E, Code, 128, 1>(p, kmap, vmap, num_sms, stream)
                    : launch<E, Code, 64, 1>(p, kmap, vmap, num_sms, stream);
  return D == 128 ? launch<E, Code, 128, 2>(p, kmap, vmap, num_sms, stream)
                  : launch<E, Code, 64, 2>(p, kmap, vmap, num_sms, stream);
}

struct Scratch {
  size_t rows, descs;
  int per_piece;
};
Scratch scratch_of(int hq, int n_kv_heads, int num_sms) {
  const int g = hq / n_kv_heads, g16 = g < 16 ? g : 16;
  const size_t ctas = 2 * static_cast<size_t>(num_sms);
  return Scratch{2 * ctas * g16, ctas, g16};
}

}  // namespace

size_t quantized_attention_workspace(int hq, int n_kv_heads, int D, int num_sms) {
  const Scratch s = scratch_of(hq, n_kv_heads, num_sms);
  // Descriptions first (16 bytes each), then the rows.
  return (s.descs * sizeof(Desc) + s.rows * (D + 2) * 4 + 255) / 256 * 256;
}

cudaError_t launch_quantized_attention(const QuantizedPool& pool, const QuantizedSeqs& seqs, const CUtensorMap& kmap,
                                       const CUtensorMap& vmap, const QuantizedAttentionArgs& a, int num_sms,
                                       cudaStream_t stream) {
  const Scratch s = scratch_of(a.hq, pool.n_kv_heads, num_sms);
  Params p = {};
  p.q = a.q;
  p.out = a.out;
  p.table = seqs.table;
  p.lens = seqs.lens;
  p.desc = static_cast<Desc*>(a.workspace);
  p.part = reinterpret_cast<float*>(p.desc + s.descs);
  p.m = p.part + s.rows * pool.D;
  p.l = p.m + s.rows;
  p.rows = s.per_piece;
  p.q_stride_seq = a.q_stride_seq;
  p.q_stride_head = a.q_stride_head;
  p.table_stride = seqs.table_stride;
  p.n_pages = pool.n_pages;
  p.B = seqs.B;
  p.hq = a.hq;
  p.hkv = pool.n_kv_heads;
  p.g = a.hq / pool.n_kv_heads;
  p.nrb = (p.g + 15) / 16;
  while ((1 << p.page_shift) < pool.page_size) ++p.page_shift;
  while ((1 << p.block_shift) < pool.block) ++p.block_shift;
  const int64_t limit = static_cast<int64_t>(seqs.table_width) * pool.page_size;
  p.len_limit = limit < (1 << 30) ? static_cast<int>(limit) : 1 << 30;
  p.scale_log2 = static_cast<float>(a.scale * 1.4426950408889634);
  p.starved = a.starved;
  p.wait_ns = a.wait_ns ? a.wait_ns : kWaitLimitNs;
  // An item's start and end, in tiles' time: 64 sequences of 900 to 16000
  // positions, 64 and 8 heads, 137 us with 1, 121 with 2 and 3, 122 with 4, 127
  // with 6; 8 sequences of 4000 of 8 heads on one 13.8 and 14.5.
  p.item_tiles = 2;
  p.n_units32 = static_cast<double>(p.B) * p.hkv * p.nrb * (p.len_limit / kTile + 2 + p.item_tiles) < 2147483648.0;
  p.k_scale = pool.k_scale;
  p.v_scale = pool.v_scale;
  p.k_open = pool.k_open;
  p.v_open = pool.v_open;
  p.open_slots = seqs.open_slots;
  p.scale_page_stride = pool.scale_page_stride;
  p.scale_head_stride = pool.scale_head_stride;
  p.open_stride = pool.open_stride;
  p.open_head_stride = pool.open_head_stride;
  p.n_open = pool.n_open;
  if (pool.bf16)
    return pool.e4m3 ? launch_for<__nv_bfloat16, E4m3>(p, pool.D, kmap, vmap, num_sms, stream)
                     : launch_for<__nv_bfloat16, Int8>(p, pool.D, kmap, vmap, num_sms, stream);
  return pool.e4m3 ? launch_for<__half, E4m3>(p, pool.D, kmap, vmap, num_sms, stream)
                   : launch_for<__half, Int8>(p, pool.D, kmap, vmap, num_sms, stream);
}

}  // namespace dqg

DQG_STATUS_READER(read_status_quantized_attention)
