// Rotation and storing of a batch of tokens in a cache held in 8 bits: queries
// as in paged_append.cu (formulas: paged_rope.cuh), keys and values in blocks
// of 16, 32 or 64 positions of one head with one fp32 scale:
//
//   x = E(rotated key) or value, in the 16-bit type E, as a 16-bit cache holds it
//   s = max(max |x| / L, 2^-126),  code = round(x / s)      (L = 127 or 448)
//
// A block is quantised once, when its last position comes: until then its rows
// wait in 16 bits in the sequence's open block. (Codes that were rounded again
// whenever a later row raises the block's maximum would save that memory and
// lose up to half a step each time, and would depend on how a prompt was cut
// into calls.) 2^-126 keeps 1 / s finite; a value that is not finite makes s
// NaN, and with it all of the block.
//
// Some blocks of the grid take queries, the others a block of positions of one
// KV head each: keys, then values, sixteen values of a row a thread.
// The block that completes a sequence's open block also stores the new open
// rows, whose place it has read before; no other reads or writes them.
//
// Bound by HBM with long batches: 8192 tokens of 64 and 8 heads of 128 with
// norms (bf16 to e4m3; 168 MB read, 151 written, 49 us at the copy rate) 65 us,
// of which the writes that stay in L2 show half (172 MB read, 96 MB written).
// Registers bound it next (29 % of the warps resident, at 96): eight heads a
// lane group one after the other took 114 us, four with passes and codes apart
// 67, keys' and values' rows loaded together 65. (Of the 30 variants the five of
// uneven rotations in two or four passes spill, 16 to 60 bytes.) With heads of 64
// and blocks of 16 half of a block's threads have no row: 1754 tokens in ragged
// chunks, of 32 and 8 such heads, take 9.9 us. Small batches are a launch: 8 tokens
// 4.3 us in a graph.
#include <cstdint>

#include "paged_rope.cuh"
#include "quantized.cuh"

namespace dqg {
namespace {

constexpr int kThreads = 128;
constexpr int kIter = 4;  // heads a lane group takes one after the other, at most

template <typename E>
struct Params {
  const E* qkv;
  const float* cosv;
  const float* sinv;
  const int64_t* positions;
  const E* q_norm;
  const E* k_norm;
  E* q_out;
  QuantizedPool pool;
  QuantizedSeqs seqs;
  int64_t qkv_stride, n_positions, q_blocks;
  int T, hq, hkv, rot, page_shift, block_shift, chunks, iter;
  float eps;
};

struct Seq {
  int q0, n, end;  // first row of qkv, new rows, length with them
};
// A sequence's rows; none where its description is out of order or range.
template <typename E>
__device__ __forceinline__ Seq load_seq(const Params<E>& p, int b, bool report) {
  Seq s;
  s.q0 = __ldg(p.seqs.q_starts + b);
  s.end = __ldg(p.seqs.lens + b);
  const int64_t n = static_cast<int64_t>(__ldg(p.seqs.q_starts + b + 1)) - s.q0;
  const int64_t limit = static_cast<int64_t>(p.seqs.table_width) << p.page_shift;
  const int slot = __ldg(p.seqs.open_slots + b);
  const bool good = s.q0 >= 0 && n >= 0 && s.q0 + n <= p.T && (n == 0 || (n <= s.end && s.end <= limit && slot >= 0 &&
                                                                          slot < p.pool.n_open));
  if (!good && report) atomicOr(&g_status, kStatusBadIndex);
  s.n = good ? static_cast<int>(n) : 0;
  return s;
}
// Blocks of positions that a sequence's new rows touch on, the open one at its
// end counted with the first.
template <typename E>
__device__ __forceinline__ uint32_t units_of(const Params<E>& p, const Seq& s) {
  if (s.n == 0) return 0;
  const int first = (s.end - s.n) >> p.block_shift, done = s.end >> p.block_shift;
  return done > first ? done - first : 1;
}

__device__ __forceinline__ int64_t clamped_position(int64_t pos, int64_t n, bool report) {
  if (pos < 0 || pos >= n) {
    if (report) atomicOr(&g_status, kStatusBadIndex);
    return pos < 0 ? 0 : n - 1;
  }
  return pos;
}

template <typename E, int D, int LAYOUT>
__device__ __forceinline__ void store_queries(const Params<E>& p, int64_t block) {
  using Lane = RopeLane<E, D, LAYOUT>;
  constexpr int kGroups = 32 / Lane::kLanes;  // heads a warp holds at a time
  const int64_t w = block * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t token = w / p.chunks;
  const int lane = threadIdx.x & 31, grp = lane / Lane::kLanes;
  const int h0 = static_cast<int>(w - token * p.chunks) * p.iter * kGroups + grp;
  if (token >= p.T) return;
  Lane part(lane % Lane::kLanes, p.rot);
  const E* row = p.qkv + token * p.qkv_stride;
  uint4 xa[kIter], xb[kIter];
#pragma unroll
  for (int it = 0; it < kIter; ++it) {
    const int h = h0 + it * kGroups;
    if (it < p.iter && h < p.hq) {
      xa[it] = __ldcs(reinterpret_cast<const uint4*>(row + static_cast<int64_t>(h) * D + part.ea));
      xb[it] = __ldcs(reinterpret_cast<const uint4*>(row + static_cast<int64_t>(h) * D + part.eb));
    }
  }
  const int64_t pos = clamped_position(__ldg(p.positions + token), p.n_positions, lane == 0);
  part.entries(p.cosv + pos * part.half, p.sinv + pos * part.half);
#pragma unroll
  for (int it = 0; it < kIter; ++it) {
    const int h = h0 + it * kGroups;
    if (it >= p.iter || h - grp >= p.hq) break;  // (by whole warps)
    float a[8], b[8];
    unpack8<E>(h < p.hq ? xa[it] : make_uint4(0, 0, 0, 0), a);
    unpack8<E>(h < p.hq ? xb[it] : make_uint4(0, 0, 0, 0), b);
    const float r = part.norm(a, b, p.q_norm, p.eps);
    if (h >= p.hq) continue;
    part.rotate(a, b, row + static_cast<int64_t>(h) * D, p.q_norm, r);
    E* dst = p.q_out + (token * p.hq + h) * D;
    __stcs(reinterpret_cast<uint4*>(dst + part.ea), pack8<E>(a));
    __stcs(reinterpret_cast<uint4*>(dst + part.eb), pack8<E>(b));
  }
}

// Largest magnitude among 16-bit values, as bits (an infinity or NaN is larger
// than any finite value).
__device__ __forceinline__ uint32_t magnitude(uint4 v, uint32_t m) {
  m = __vmaxu2(m, v.x & 0x7fff7fffu);
  m = __vmaxu2(m, v.y & 0x7fff7fffu);
  m = __vmaxu2(m, v.z & 0x7fff7fffu);
  return __vmaxu2(m, v.w & 0x7fff7fffu);
}

// kPasses: a block's rows over those that the threads hold at a time.
template <typename E, int D, int LAYOUT, int kPasses>
__device__ __forceinline__ void store_block(const Params<E>& p, int b, const Seq& s, int j, int kvh, uint32_t* scratch) {
  using Lane = RopeLane<E, D, LAYOUT>;
  constexpr int kRows = kThreads / Lane::kLanes;       // rows at a time
  const int row0 = threadIdx.x / Lane::kLanes;
  const int base = j << p.block_shift, block = 1 << p.block_shift, start = s.end - s.n;
  const bool whole = base + block <= s.end;
  const int64_t slot = __ldg(p.seqs.open_slots + b);
  int page = whole ? __ldg(p.seqs.table + b * p.seqs.table_stride + (base >> p.page_shift)) : 0;
  if (page < 0 || page >= p.pool.n_pages) {
    if (threadIdx.x == 0) atomicOr(&g_status, kStatusBadIndex);
    page = -1;
  }
  // Rows of both, all loads ahead of the first use (8192 tokens 66.8 -> 64.9 us).
  uint4 xa[2][kPasses], xb[2][kPasses];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const E* open = static_cast<const E*>(which ? p.pool.v_open : p.pool.k_open) + slot * p.pool.open_stride +
                    kvh * p.pool.open_head_stride;
    const Lane part(threadIdx.x % Lane::kLanes, which ? 0 : p.rot);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      xa[which][i] = xb[which][i] = make_uint4(0, 0, 0, 0);
      const int row = row0 + i * kRows, t = base + row;
      if (row < block && t >= start && t < s.end) {
        const E* head = p.qkv + (s.q0 + t - start) * p.qkv_stride +
                        static_cast<int64_t>(p.hq + (which ? p.hkv : 0) + kvh) * D;
        xa[which][i] = __ldcs(reinterpret_cast<const uint4*>(head + part.ea));
        xb[which][i] = __ldcs(reinterpret_cast<const uint4*>(head + part.eb));
      } else if (whole && row < block && t < start) {  // stored by an earlier call
        xa[which][i] = *reinterpret_cast<const uint4*>(open + row * D + part.ea);
        xb[which][i] = *reinterpret_cast<const uint4*>(open + row * D + part.eb);
      }
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = row0 + i * kRows, t = base + row;
      const bool fresh = row < block && t >= start && t < s.end;
      Lane part(threadIdx.x % Lane::kLanes, which ? 0 : p.rot);
      if (!which) {
        const int64_t token = s.q0 + (fresh ? t - start : 0);
        const int64_t pos = clamped_position(__ldg(p.positions + token), p.n_positions, false);
        part.entries(p.cosv + pos * part.half, p.sinv + pos * part.half);
        float x[8], y[8];
        unpack8<E>(xa[0][i], x);
        unpack8<E>(xb[0][i], y);
        const float r = part.norm(x, y, p.k_norm, p.eps);
        if (fresh) {
          part.rotate(x, y, p.qkv + token * p.qkv_stride + static_cast<int64_t>(p.hq + kvh) * D, p.k_norm, r);
          xa[0][i] = pack8<E>(x);
          xb[0][i] = pack8<E>(y);
        }
      }
      if (!whole && fresh) {
        E* open = static_cast<E*>(which ? p.pool.v_open : p.pool.k_open) + slot * p.pool.open_stride +
                  kvh * p.pool.open_head_stride + row * D;
        *reinterpret_cast<uint4*>(open + part.ea) = xa[which][i];
        *reinterpret_cast<uint4*>(open + part.eb) = xb[which][i];
      }
      most = magnitude(xb[which][i], magnitude(xa[which][i], most));
    }
    if (!whole) continue;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, off));
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) most = __vmaxu2(most, scratch[w]);
    __syncthreads();
    const float2 two = Elem<E>::unpack(most);
    const bool finite = Elem<E>::non_finite(most) == 0u;
    const bool e4m3 = p.pool.e4m3;
    // code = round(x / s), formed as (L x) / max |x|: the product is exact, and
    // the quotient too where it is a number of few bits (a reciprocal's product,
    // and one Newton step on the quotient), so that a value halfway between two
    // codes is seen to be. Without that 1.5 times the rounding errors of codes,
    // with a division 73 instead of 67 us for 8192 tokens.
    const float largest = fmaxf(two.x, two.y), range = e4m3 ? E4m3::kMost : Int8::kMost;
    const bool tiny = largest / range < 1.17549435e-38f;
    const float scale = finite ? (tiny ? 1.17549435e-38f : largest / range) : NAN;
    // (Large values by 2^-64 of themselves: bf16's largest times L is no number.)
    const float less = largest > 1e30f ? 5.42101086e-20f : 1.f;
    const float up = tiny ? 8.50705917e37f : range * less, down = tiny ? 1.f : largest * less, inv = 1.f / down;  // (2^126)
    if (page < 0) continue;
    if (threadIdx.x == 0) {
      float* to = (which ? p.pool.v_scale : p.pool.k_scale) + page * p.pool.scale_page_stride +
                  kvh * p.pool.scale_head_stride;
      to[(base & ((1 << p.page_shift) - 1)) >> p.block_shift] = scale;
    }
    uint8_t* codes = static_cast<uint8_t*>(which ? p.pool.v : p.pool.k) + page * p.pool.page_stride +
                     kvh * p.pool.head_stride + (base & ((1 << p.page_shift) - 1)) * p.pool.row_stride;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = row0 + i * kRows;
      if (row >= block) continue;
      const Lane part(threadIdx.x % Lane::kLanes, which ? 0 : p.rot);
      float x[8];
#pragma unroll
      for (int run = 0; run < 2; ++run) {
        unpack8<E>(run ? xb[which][i] : xa[which][i], x);
        uint2 w = make_uint2(0, 0);
        if (finite) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float t = x[e] * up, y = t * inv;
            x[e] = fmaf(fmaf(-y, down, t), inv, y);
          }
          w = e4m3 ? make_uint2(E4m3::pack4(x[0], x[1], x[2], x[3]), E4m3::pack4(x[4], x[5], x[6], x[7]))
                   : make_uint2(Int8::pack4(x[0], x[1], x[2], x[3]), Int8::pack4(x[4], x[5], x[6], x[7]));
        }
        __stcs(reinterpret_cast<uint2*>(codes + row * p.pool.row_stride + (run ? part.eb : part.ea)), w);
      }
    }
  }
}

template <typename E, int D, int LAYOUT, int kPasses>
__global__ void __launch_bounds__(kThreads, kPasses == 4 ? 3 : (LAYOUT == kUneven ? 4 : 5))
    quantized_append_kernel(const __grid_constant__ Params<E> p) {
  __shared__ uint32_t scratch[kThreads / 32 + 2];
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  // (Keys and values first: their blocks take longer, and the queries' fill up
  // behind them.)
  const int64_t kv_blocks = gridDim.x - p.q_blocks, u = blockIdx.x;
  if (u >= kv_blocks) {
    store_queries<E, D, LAYOUT>(p, u - kv_blocks);
    return;
  }
  const int kvh = static_cast<int>(u % p.hkv);
  int64_t in = 0;
  // (The last unit is behind all others: it looks at every sequence.)
  const bool report = u == kv_blocks - 1;
  const int b = find_unit(p.seqs.B, u / p.hkv, [&](int i) { return units_of(p, load_seq(p, i, report)); }, scratch, &in);
  if (b < 0) return;
  const Seq s = load_seq(p, b, false);
  const int first = (s.end - s.n) >> p.block_shift, last = (s.end - 1) >> p.block_shift;
  __syncthreads();
  store_block<E, D, LAYOUT, kPasses>(p, b, s, first + static_cast<int>(in), kvh, scratch);
  if (in == 0 && last > first && (s.end & ((1 << p.block_shift) - 1))) {
    __syncthreads();  // the open rows have been read
    store_block<E, D, LAYOUT, kPasses>(p, b, s, last, kvh, scratch);
  }
}

template <typename E, int D, int kPasses>
cudaError_t launch(const QuantizedPool& pool, const QuantizedSeqs& seqs, const QuantizedAppendArgs& a, int num_sms,
                   cudaStream_t stream) {
  Params<E> p;
  p.qkv = static_cast<const E*>(a.qkv);
  p.cosv = a.cosv;
  p.sinv = a.sinv;
  p.positions = a.positions;
  p.q_norm = static_cast<const E*>(a.q_norm);
  p.k_norm = static_cast<const E*>(a.k_norm);
  p.q_out = static_cast<E*>(a.q_out);
  p.pool = pool;
  p.seqs = seqs;
  p.qkv_stride = a.qkv_stride;
  p.n_positions = a.n_positions;
  p.T = a.T;
  p.hq = a.hq;
  p.hkv = pool.n_kv_heads;
  p.rot = a.rot;
  p.eps = a.eps;
  p.page_shift = p.block_shift = 0;
  while ((1 << p.page_shift) < pool.page_size) ++p.page_shift;
  while ((1 << p.block_shift) < pool.block) ++p.block_shift;
  // kIter heads a lane group once that still fills the GPU's warps; below it
  // one, so that a few tokens spread over the SMs.
  constexpr int kGroups = 32 / (D / 16);
  p.iter = static_cast<int64_t>(a.T) * a.hq / kGroups >= kIter * 64 * static_cast<int64_t>(num_sms) ? kIter : 1;
  p.chunks = (a.hq + kGroups * p.iter - 1) / (kGroups * p.iter);
  p.q_blocks = (static_cast<int64_t>(a.T) * p.chunks + kThreads / 32 - 1) / (kThreads / 32);
  // n new rows make (n - 1) / block + 1 units at most; and one more than all.
  const int64_t units = a.T / pool.block + (a.T < seqs.B ? a.T : seqs.B) + 1;
  const int64_t blocks = p.q_blocks + units * pool.n_kv_heads;
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
  if (a.interleaved) return cudaLaunchKernelEx(&cfg, quantized_append_kernel<E, D, kInterleaved, kPasses>, p);
  if (a.rot % 16 == 0) return cudaLaunchKernelEx(&cfg, quantized_append_kernel<E, D, kHalf, kPasses>, p);
  return cudaLaunchKernelEx(&cfg, quantized_append_kernel<E, D, kUneven, kPasses>, p);
}

template <typename E, int D>
cudaError_t launch_passes(const QuantizedPool& pool, const QuantizedSeqs& seqs, const QuantizedAppendArgs& a, int num_sms,
                          cudaStream_t stream) {
  const int rows = kThreads / (D / 16);  // that the threads hold at a time
  if (pool.block <= rows) return launch<E, D, 1>(pool, seqs, a, num_sms, stream);
  if (pool.block <= 2 * rows) return launch<E, D, 2>(pool, seqs, a, num_sms, stream);
  if constexpr (D == 128) return launch<E, D, 4>(pool, seqs, a, num_sms, stream);
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_quantized_append(const QuantizedPool& pool, const QuantizedSeqs& seqs, const QuantizedAppendArgs& a,
                                    int num_sms, cudaStream_t stream) {
  if (pool.bf16)
    return pool.D == 128 ? launch_passes<__nv_bfloat16, 128>(pool, seqs, a, num_sms, stream)
                         : launch_passes<__nv_bfloat16, 64>(pool, seqs, a, num_sms, stream);
  return pool.D == 128 ? launch_passes<__half, 128>(pool, seqs, a, num_sms, stream)
                       : launch_passes<__half, 64>(pool, seqs, a, num_sms, stream);
}

}  // namespace dqg

DQG_STATUS_READER(read_status_quantized_append)
