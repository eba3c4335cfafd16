// Decode attention over a paged cache: one query token per sequence, lengths
// on the device, grouped KV heads. No reference counterpart (the reference
// models the cache's bytes, dequant/byte_model.py:214-219).
//
//   o[b, h] = softmax(scale q[b, h] . K_b[:, h / g]^T) V_b[:, h / g]
//
// over the lens[b] positions that sequence b's pages hold; zero where there is
// none. Every key and value row is read once for every 16 query heads of its KV
// head (8 times at most, by CTAs that share the L2 cache), so HBM bounds it up to
// 16: 32 sequences of 4000 positions and one KV head take 21 us with 16 query
// heads, 28 with 32, 74 with 128 (65 MB, 10 us at the copy rate).
//
// Work is counted in tiles of 64 positions, sequence by sequence and KV head
// by KV head, and cut into equal shares, one per CTA (two CTAs per SM), so that
// lengths of any spread keep every SM streaming to the end; the shares follow
// from the lengths on the device, so a captured launch serves other lengths.
// In a CTA one warp copies the tiles' page rows into a ring in shared memory
// (tensor-map boxes of whole page rows, 128-byte swizzle) and four warps take
// 16 positions of a tile each: S^T = Q K^T by mma.m16n8k16 with the KV head's
// query heads as the A rows, online softmax in fp32, O += P V with P (16-bit,
// as the values are) from the score registers. An item (sequence, head) that
// lies in one share is finished by its CTA; one that is cut leaves a (max, sum,
// O) piece per CTA in the workspace, and a second small kernel joins the
// pieces in order. No atomics: the same lengths give the same bits. Behind a
// shared prefix every item leaves its result to the second kernel, which joins
// it with the prefix's pieces: nothing here waits for those.
//
// Waits are bounded. A consumer warp whose wait ran out goes on through its
// items without data and makes their results NaN, so that the barriers among
// the warps are always met and every item is described to the second kernel.
//
// A prefix whose rows (sequences times query heads of a KV head) fit one or two
// 16-row tiles is streamed by this kernel itself, as items of its own ahead of the
// sequences' (prefix_streamed below); one with more rows is left to the prompt
// kernel, which reads it once for 256 rows.
//
// Measured (B200, a stream of calls whose inputs alternate between three sets):
// 64 sequences of 900 to 16000 positions, 64 query and 8 KV heads, bf16, 1.25 GB:
// 206 us, 6.08 TB/s, 0.94 of the rate that a copy reaches (both kernels; the first
// alone 200 us, 6.27); HBM bounds it. Short calls are bound by latency: one
// sequence of 2049 positions, 32 heads (33.5 MB): 13 us (12.4 replayed from a
// graph), about 4 of them before the first tile has come (shares, table, copies),
// 4.5 streaming, 3 for the second kernel.
#include <cstdint>

#include "paged_decode.cuh"

namespace dqg {
namespace {

constexpr int kTile = 64;              // positions per tile
constexpr int kWarps = 4;              // consumer warps
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kStages = 3;
constexpr int kCtasPerSm = 2;
constexpr int kQuerySlots = 4;         // items whose queries are held at most
constexpr int kMergeRows = 4;          // query heads per round of the warps' merge
// Weights are formed for the values' 16-bit type, relative to a reference 2^15
// below the running maximum: of fp16's range (2^-24 to 2^16) all that lies above
// 1 is used too, so that what a weight loses at the lower end is below 2^-40 of
// the largest one. References are in log2 units, and with every piece its own.
// (One rounding of a weight, to the type that the product's two operands share,
// adds up to a quarter to the output's own error. Weights as a sum of two 16-bit
// numbers and a second product left the output's alone: large batches took the
// same 201 us, but short calls 12.9 us instead of 12.3, small prefixes 25.6
// instead of 24.3.)
constexpr float kHeadroom = 15.f;

using Params = DecodeParams;

__device__ __forceinline__ int tiles_of(const Params&, int len) { return len > 0 ? (len + kTile - 1) / kTile : 1; }

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile: halves of 64
// values, 128-byte rows, swizzled as the tensor map writes them.
__device__ __forceinline__ uint32_t tile_off(int row, int chunk) {
  return static_cast<uint32_t>((chunk >> 3) * (kTile * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

template <int D>
struct Layout {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kRing = kStages * 2 * kTileBytes;
  static constexpr int kMerge = kWarps * kMergeRows * D * 4;
  static constexpr int kQuery = 16 * D * 2;
  static constexpr int kSmem = 1024 + kRing + kMerge + kQuery + kWarps * 16 * 8 + 2 * (kStages + kQuerySlots + 1) * 8 + 80;
};

template <typename E, int D>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    paged_decode_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap) {
  using L = Layout<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  // Queries of the items ahead; reads of 16 rows run past a short slot, at
  // worst into the merge buffer (rows whose results nobody takes).
  uint8_t* qs = smem + L::kRing;
  float* os = reinterpret_cast<float*>(qs + L::kQuery);               // [warp][4][D]
  float* ms = os + L::kMerge / 4;                                     // [warp][16]
  float* ls = ms + kWarps * 16;
  uint64_t* full = reinterpret_cast<uint64_t*>(ls + kWarps * 16);
  uint64_t* empty = full + kStages;
  uint64_t* q_full = empty + kStages;
  uint64_t* q_empty = q_full + kQuerySlots;
  uint64_t* pre_full = q_empty + kQuerySlots;  // a streamed prefix's queries take all slots
  uint64_t* pre_empty = pre_full + 1;
  Share* share = reinterpret_cast<Share*>(pre_empty + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, kWarps);
    }
    for (int i = 0; i < kQuerySlots; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, kWarps);
    }
    mbar_init(pre_full, 1);
    mbar_init(pre_empty, kWarps);
    fence_mbar_init();
    tma_prefetch_map(&kmap);
    tma_prefetch_map(&vmap);
  }
  // Rows that no query head fills stay zero.
  for (int i = threadIdx.x; i < L::kQuery / 16; i += kThreads) reinterpret_cast<uint4*>(qs)[i] = make_uint4(0, 0, 0, 0);
  fence_async_shared();
  // After a prefix kernel (which every one of its CTAs lets this one start
  // from only once its own inputs are complete), the queries, pages and
  // lengths may be read at once; only the end waits (and with it everything
  // behind this kernel).
  const bool late = p.prefix.S > 0;
  const bool joined = late || p.pre_items > 0;  // results are joined with a prefix's
  if (!late) pdl_wait_prior_grid();
  if (warp == 0) {
    const Share s = find_share(p, blockIdx.x, gridDim.x);
    if (lane == 0) *share = s;
  }
  __syncthreads();
  pdl_launch_dependents();
  Share s = *share;
  const int q_rows = min(16, p.g), q_slots = min(kQuerySlots, 16 / q_rows);

  if (warp == kWarps) {
    // ---- the copying warp: 16-row (or box_rows-row) pieces of page rows.
    const int per = p.box_rows;                 // rows a box
    const int boxes = kTile / per * (D / 64);   // K boxes a tile; as many V boxes
    const int my = lane, half = my % (D / 64), sub = my / (D / 64);
    const uint64_t policy = policy_evict_last();
    int it = 0, item = 0, pre = 0;
    bool ok = !(p.starved >> kWarps & 1);
    while (s.count > 0 && ok) {
      const Item i = item_of(p, s);
      if (i.x1 == i.x0) {  // the cut falls before its first tile
        advance(p, s, i.units);
        continue;
      }
      // The item's queries, a row a lane.
      if (s.b < 0) {
        if (pre > 0 && !warp_wait(pre_empty, (pre - 1) & 1, p.wait_ns)) break;
        if (lane == 0) mbar_arrive_expect_tx(pre_full, i.rows * D * 2);
        __syncwarp();
        if (lane < i.rows)
          bulk_g2s(qs + lane * D * 2, static_cast<const E*>(p.q) + (i.first + lane / p.g) * p.q_stride_seq +
                   (i.head0 + lane % p.g) * p.q_stride_head, D * 2, pre_full, policy);
        ++pre;
      } else {
        if (lane == 0 && __ldg(p.lens + s.b) != i.len) atomicOr(&g_status, kStatusBadIndex);
        if (item == 0 && pre > 0 && !warp_wait(pre_empty, (pre - 1) & 1, p.wait_ns)) break;
        const int qi = item % q_slots;
        if (item >= q_slots && !warp_wait(q_empty + qi, ((item / q_slots) & 1) ^ 1, p.wait_ns)) break;
        if (lane == 0) mbar_arrive_expect_tx(q_full + qi, i.rows * D * 2);
        __syncwarp();
        if (lane < i.rows)
          bulk_g2s(qs + (qi * q_rows + lane) * D * 2, static_cast<const E*>(p.q) + s.b * p.q_stride_seq +
                   (i.head0 + lane) * p.q_stride_head, D * 2, q_full + qi, policy);
        ++item;
      }
      for (int x = i.x0; x < i.x1; ++x, ++it) {
        const int st = it % kStages;
        const int t = x * kTile + sub * per;
        int page = static_cast<int>(p.n_pages);  // no such page: zeros
        if (my < boxes && t < i.len) {
          page = __ldg(i.table + (t >> p.page_shift));
          if (page < 0 || page >= p.n_pages) {
            page = static_cast<int>(p.n_pages);
            atomicOr(&g_status, kStatusBadIndex);
          }
        }
        if (it >= kStages && !warp_wait(empty + st, ((it / kStages) & 1) ^ 1, p.wait_ns)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(full + st, 2 * L::kTileBytes);
        __syncwarp();
        if (my < boxes) {
          const uint32_t dst = smem_u32(smem) + st * 2 * L::kTileBytes + half * (kTile * 128) + sub * per * 128;
          const int in_page = t & ((1 << p.page_shift) - 1);
          tma_load_4d(dst, &kmap, full + st, half * 64, in_page, i.kvh, page);
          tma_load_4d(dst + L::kTileBytes, &vmap, full + st, half * 64, in_page, i.kvh, page);
        }
      }
      advance(p, s, i.units);
    }
    // Copies still in flight land before the CTA's memory goes (bounded).
    if (pre > 0) warp_wait(pre_full, (pre - 1) & 1, p.wait_ns);
    for (int i = item < q_slots ? 0 : item - q_slots; i < item; ++i)
      if (!warp_wait(q_full + i % q_slots, (i / q_slots) & 1, p.wait_ns)) break;
    for (int i = it < kStages ? 0 : it - kStages; i < it; ++i)
      if (!warp_wait(full + i % kStages, (i / kStages) & 1, p.wait_ns)) break;
  } else {
    const int gid = lane >> 2, c = lane & 3;
    const uint32_t ring = smem_u32(smem);
    const int p0 = warp * 16;
    int it = 0, item = 0, pre = 0;
    // Once a wait has run out no later one is taken.
    bool ok = !(p.starved >> warp & 1), cut_first = false;
    auto await = [&](uint64_t* bar, uint32_t parity) { return ok = ok && warp_wait(bar, parity, p.wait_ns); };
    while (s.count > 0) {
      const Item i = item_of(p, s);
      const int len = i.len, head0 = i.head0, rows = i.rows;
      if (i.x1 == i.x0) {
        advance(p, s, i.units);
        continue;
      }
      // Q as A fragments: rows are the KV head's query heads (of several
      // sequences, in a prefix).
      uint32_t qa[D / 16][4];
      const int qi = s.b < 0 ? 0 : item % q_slots;
      await(s.b < 0 ? pre_full : q_full + qi, (s.b < 0 ? pre : item / q_slots) & 1);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
        ldsm_x4(smem_u32(qs) + (qi * q_rows + (lane & 15)) * (D * 2) + ks * 32 + (lane >> 4) * 16, qa[ks]);
      float o[D / 8][4];
#pragma unroll
      for (int nb = 0; nb < D / 8; ++nb) o[nb][0] = o[nb][1] = o[nb][2] = o[nb][3] = 0.f;
      float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
      for (int x = i.x0; x < i.x1; ++x, ++it) {
        const int st = it % kStages;
        if (!await(full + st, (it / kStages) & 1)) continue;
        const uint32_t kst = ring + st * 2 * L::kTileBytes, vst = kst + L::kTileBytes;
        const int ts = x * kTile + p0;
        if (ts < len) {
          if (ts + 16 > len) {
            // The last page's rows behind the sequence's end hold anything:
            // zero this warp's part of their values (a zero weight times an
            // infinity would not be zero).
            for (int i = lane; i < 16 * (D / 8); i += 32) {
              const int r = i / (D / 8), ch = i % (D / 8);
              if (ts + r >= len)
                *reinterpret_cast<uint4*>(smem + (vst - ring) + tile_off(p0 + r, ch)) = make_uint4(0, 0, 0, 0);
            }
            fence_async_shared();  // before the ring's next copy to this place
            __syncwarp();
          }
          float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t b[4];
            ldsm_x4(kst + tile_off(p0 + ((lane >> 4) & 1) * 8 + (lane & 7), ks * 2 + ((lane >> 3) & 1)), b);
            Elem<E>::mma(sc[0], qa[ks], b[0], b[1]);
            Elem<E>::mma(sc[1], qa[ks], b[2], b[3]);
          }
          float pr[2][4];
#pragma unroll
          for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = ts + nb * 8 + 2 * c + (e & 1);
              sc[nb][e] = t < len ? sc[nb][e] * p.scale_log2 : -INFINITY;
            }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float mx = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m_run[r], mx);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float corr = exp2_approx(m_run[r] - m_use), ref = m_use - kHeadroom;
            l_run[r] *= corr;
#pragma unroll
            for (int nb = 0; nb < D / 8; ++nb) {
              o[nb][2 * r] *= corr;
              o[nb][2 * r + 1] *= corr;
            }
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
              pr[nb][2 * r] = exp2_approx(sc[nb][2 * r] - ref);
              pr[nb][2 * r + 1] = exp2_approx(sc[nb][2 * r + 1] - ref);
              l_run[r] += pr[nb][2 * r] + pr[nb][2 * r + 1];
            }
            m_run[r] = m_new;
          }
          uint32_t pa[4];
          pa[0] = Elem<E>::pack(pr[0][0], pr[0][1]);
          pa[1] = Elem<E>::pack(pr[0][2], pr[0][3]);
          pa[2] = Elem<E>::pack(pr[1][0], pr[1][1]);
          pa[3] = Elem<E>::pack(pr[1][2], pr[1][3]);
#pragma unroll
          for (int dp = 0; dp < D / 16; ++dp) {
            uint32_t b[4];
            ldsm_x4_trans(vst + tile_off(p0 + ((lane >> 3) & 1) * 8 + (lane & 7), dp * 2 + ((lane >> 4) & 1)), b);
            Elem<E>::mma(o[2 * dp], pa, b[0], b[1]);
            Elem<E>::mma(o[2 * dp + 1], pa, b[2], b[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + st);
      }
      // The queries' place is free once their reads have come back, not once
      // they are issued: here every fragment is used (by the products, or, in a
      // warp whose slices all lay behind the end, by this).
      if (i.x0 * kTile + p0 >= len) {
        uint32_t x = 0;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) x ^= qa[ks][0] ^ qa[ks][1] ^ qa[ks][2] ^ qa[ks][3];
        asm volatile("" ::"r"(x) : "memory");
      }
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(s.b < 0 ? pre_empty : q_empty + qi);
      if (s.b < 0) ++pre;
      else ++item;

      // The item's (or piece's) result: the warps' parts, four heads a round.
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
        if (c == 0) {
          ms[warp * 16 + gid + 8 * r] = m_run[r] - kHeadroom;
          ls[warp * 16 + gid + 8 * r] = ok ? l_run[r] : NAN;
        }
      }
      const bool whole = i.x0 == 0 && i.x1 == i.tiles;
      const int64_t row0 = whole ? whole_row(p, s.b, s.hv)
                                 : (2 * static_cast<int64_t>(blockIdx.x) + (i.x0 > 0 ? 0 : 1)) * p.rows;
      if (i.x0 == 0 && (joined || !whole)) {
        cut_first = true;
        if (threadIdx.x == 0) {
          const int64_t items = static_cast<int64_t>(p.B) * p.hkv * p.nrb;
          const int64_t id = s.b < 0 ? items + s.hv : static_cast<int64_t>(s.b) * p.hkv * p.nrb + s.hv;
          const int last = s.all.holder(s.pos - s.x + i.tiles + p.item_tiles - 1);
          p.desc[joined ? id : blockIdx.x] =
              Desc{s.b, s.hv, whole ? -1 : static_cast<int>(blockIdx.x), last - static_cast<int>(blockIdx.x) + 1};
        }
      }
      for (int r0 = 0; r0 < rows; r0 += kMergeRows) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int j = gid + 8 * r - r0;
          if (j >= 0 && j < kMergeRows)
#pragma unroll
            for (int nb = 0; nb < D / 8; ++nb)
              *reinterpret_cast<float2*>(os + (warp * kMergeRows + j) * D + nb * 8 + 2 * c) =
                  make_float2(o[nb][2 * r], o[nb][2 * r + 1]);
        }
        named_sync(1, 32 * kWarps);
        for (int i = threadIdx.x; i < kMergeRows * (D / 4); i += 32 * kWarps) {
          const int j = i / (D / 4), d4 = i % (D / 4), row = r0 + j;
          if (row < rows) {
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ms[w * 16 + row]);
            const float mu = mx == -INFINITY ? 0.f : mx;
            float den = 0.f;
            float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              const float f = exp2_approx(ms[w * 16 + row] - mu);
              const float4 v = *reinterpret_cast<const float4*>(os + (w * kMergeRows + j) * D + d4 * 4);
              den = fmaf(ls[w * 16 + row], f, den);
              num.x = fmaf(v.x, f, num.x);
              num.y = fmaf(v.y, f, num.y);
              num.z = fmaf(v.z, f, num.z);
              num.w = fmaf(v.w, f, num.w);
            }
            if (whole && !joined) {
              store4<E, D>(p, s.b, head0 + row, d4, den, num);
            } else {
              *reinterpret_cast<float4*>(p.part + (row0 + row) * D + d4 * 4) = num;
              if (d4 == 0) {
                p.m[row0 + row] = mx;
                p.l[row0 + row] = den;
              }
            }
          }
        }
        named_sync(1, 32 * kWarps);
      }
      advance(p, s, i.units);
    }
    if (threadIdx.x == 0 && !cut_first && !joined) p.desc[blockIdx.x] = Desc{0, 0, 0, 0};
  }
  if (late) pdl_wait_prior_grid();
}

template <typename E, int D>
cudaError_t launch(const Params& p, const CUtensorMap& kmap, const CUtensorMap& vmap, int num_sms,
                   cudaStream_t stream) {
  static int configured[64] = {0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(paged_decode_kernel<E, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Layout<D>::kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = 1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCtasPerSm * num_sms);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Layout<D>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, paged_decode_kernel<E, D>, p, kmap, vmap);
  if (e != cudaSuccess) return e;
  return launch_join<E, D>(p, cfg);
}

}  // namespace

int paged_decode_box_rows(int page_size) { return page_size < kTile ? page_size : kTile; }

namespace {
// What a launch leaves between its kernels: rows of pieces and whole results,
// and descriptions (see Params).
struct Scratch {
  size_t rows, descs;
  int per_piece, pre_items, pre_seqs;
};
Scratch scratch_of(int B, int hq, int n_kv_heads, int D, int prefix_len, int num_sms) {
  const int g = hq / n_kv_heads, g16 = g < 16 ? g : 16;
  const size_t items = static_cast<size_t>(B) * n_kv_heads * ((g + 15) / 16);
  const size_t ctas = static_cast<size_t>(kCtasPerSm) * num_sms;
  Scratch s{2 * ctas * g16, ctas, g16, 0, 1};
  if (prefix_len > 0) {
    if (prefix_streamed(B, hq, n_kv_heads, D, prefix_len)) {
      s.pre_seqs = 16 / g;
      s.pre_items = (B + s.pre_seqs - 1) / s.pre_seqs * n_kv_heads;
      s.per_piece = 16;
      s.rows = 2 * ctas * 16 + static_cast<size_t>(s.pre_items) * 16;
    }
    s.rows += items * g16;
    s.descs = items + s.pre_items;
  }
  return s;
}
}  // namespace

// One 16-row tile, or two of a prefix of up to 96 MiB: streaming the prefix once
// or twice beats the prompt kernel's start and its mostly empty 128-row tiles,
// until the second reading costs more. Streamed and by the prompt kernel, 32 query
// and KV heads: 16 sequences behind 2000 positions 24.2 and 34.5 us, behind 16000
// 58.4 and 71.1; 32 sequences (two tiles) behind 2000 (33 MB) 35.4 and 42.7, but
// behind 16000 (262 MB) 98.6 and 81.9. 64 and 8 heads, 4 sequences (two tiles):
// behind 2000 12.8 and 15.5, behind 16000 (66 MB) 26.6 and 30.7; four tiles behind
// 16000 39.1 and 31.3.
bool prefix_streamed(int n_seqs, int hq, int n_kv_heads, int D, int prefix_len) {
  const int g = hq / n_kv_heads;
  if (g > 16) return false;
  const int64_t bytes = static_cast<int64_t>(prefix_len) * n_kv_heads * D * 4;
  return n_seqs <= (bytes <= (int64_t(96) << 20) ? 2 : 1) * (16 / g);
}

size_t paged_decode_workspace(int B, int hq, int n_kv_heads, int D, int prefix_len, int num_sms) {
  const Scratch s = scratch_of(B, hq, n_kv_heads, D, prefix_len, num_sms);
  // Descriptions first (16 bytes each), then the rows.
  return (s.descs * sizeof(Desc) + s.rows * (D + 2) * 4 + 255) / 256 * 256;
}

cudaError_t launch_paged_decode(const PagedPool& pool, const CUtensorMap& kmap,
                                const CUtensorMap& vmap, const DecodeArgs& a, int num_sms,
                                cudaStream_t stream) {
  const Scratch s = scratch_of(a.B, a.hq, pool.n_kv_heads, pool.D, a.prefix_len, num_sms);
  Params p;
  p.q = a.q;
  p.out = a.out;
  p.table = a.table;
  p.lens = a.lens;
  p.desc = static_cast<Desc*>(a.workspace);
  p.part = reinterpret_cast<float*>(p.desc + s.descs);
  p.m = p.part + s.rows * pool.D;
  p.l = p.m + s.rows;
  p.rows = s.per_piece;
  p.pre_table = a.prefix_table;
  p.pre_len = a.prefix_len;
  p.pre_seqs = s.pre_seqs;
  p.pre_items = s.pre_items;
  p.pre_tiles = s.pre_items ? (a.prefix_len + kTile - 1) / kTile : 0;
  p.n_ctas = kCtasPerSm * num_sms;
  p.q_stride_seq = a.q_stride_seq;
  p.q_stride_head = a.q_stride_head;
  p.table_stride = a.table_stride;
  p.n_pages = pool.n_pages;
  p.B = a.B;
  p.hq = a.hq;
  p.hkv = pool.n_kv_heads;
  p.g = a.hq / pool.n_kv_heads;
  p.nrb = (p.g + 15) / 16;
  p.page_shift = 0;
  while ((1 << p.page_shift) < pool.page_size) ++p.page_shift;
  const int64_t limit = static_cast<int64_t>(a.table_width) * pool.page_size;
  p.len_limit = limit < (1 << 30) ? static_cast<int>(limit) : 1 << 30;
  p.box_rows = paged_decode_box_rows(pool.page_size);
  p.scale_log2 = a.scale_log2;
  p.starved = a.starved;
  p.wait_ns = a.wait_ns ? a.wait_ns : kWaitLimitNs;
  // With more query heads the warps' merge takes more rounds: 128 sequences of 8
  // heads a KV head behind a prefix 116 us with 1, 111 with 2, 108.5 with 3; 32 of
  // 16 heads, 4000 positions, 22.1 with 1, 21.2 with 3; 64 of 8 heads, 900 to 16000
  // positions, 202.1 and 201.6. (One the other way: 128 of 8 heads, 700 positions,
  // 18.3 and 19.2. With one head a KV head both within 2 %.)
  p.item_tiles = p.g > kMergeRows ? 3 : 1;
  p.n_units32 = static_cast<double>(a.B) * p.hkv * p.nrb * (p.len_limit / kTile + 2 + p.item_tiles) +
                    static_cast<double>(p.pre_items) * (p.pre_tiles + p.item_tiles) < 2147483648.0;
  p.prefix = a.prefix;
  if (pool.bf16)
    return pool.D == 128 ? launch<__nv_bfloat16, 128>(p, kmap, vmap, num_sms, stream)
                         : launch<__nv_bfloat16, 64>(p, kmap, vmap, num_sms, stream);
  return pool.D == 128 ? launch<__half, 128>(p, kmap, vmap, num_sms, stream)
                       : launch<__half, 64>(p, kmap, vmap, num_sms, stream);
}

}  // namespace dqg

DQG_STATUS_READER(read_status_paged_decode)
