// What the kernels of decode attention over pages share (paged_attention.cu,
// quantized_attention.cu): how a call's work is cut into equal shares, one a
// CTA, and the second kernel, which joins the pieces of the items that were
// cut. Work is counted in tiles of positions, sequence by sequence and KV head
// by KV head; a kernel's parameters derive from DecodeParams, and its
// tiles_of(p, len) says how many tiles a sequence takes.
#pragma once

#include "paged.cuh"

namespace dqg {
namespace {

struct Desc {    // an item that is joined later
  int b, hv;     // sequence, KV head and 16-row block of its query heads
  int cta;       // holds the first piece; below 0: the result lies whole in the item's own slot
  int pieces;    // 0: nothing to join
};

struct DecodeParams {
  static constexpr bool kPrefix = true;  // whether a call may have a shared prefix
  const void* q;
  void* out;
  const int32_t* table;
  const int32_t* lens;
  float* part;   // [row][D]: two pieces of `rows` rows a CTA, then (behind a prefix) whole results
  float* m;      // [row]: reference of the weights (log2 units)
  float* l;      // [row]: sum
  Desc* desc;    // [CTA]; behind a prefix [item], then [prefix item]
  const int32_t* pre_table;
  int64_t q_stride_seq, q_stride_head, table_stride, n_pages;
  int B, hq, hkv, g, nrb, rows, page_shift, len_limit, box_rows, n_ctas;
  int item_tiles;                                // an item's start and end, in tiles' time
  int pre_len, pre_seqs, pre_tiles, pre_items;  // a streamed prefix: sequences an item; tiles; items
  float scale_log2;
  uint32_t starved;  // see DecodeArgs
  uint64_t wait_ns;
  bool n_units32;   // the units of any lengths fit 31 bits
  PrefixPieces prefix;
};

// Row of a prefix piece that holds query head j of KV head `kvh` in sequence
// b, and the first of the item's pieces (layout of prompt_attention.cu).
__device__ __forceinline__ int64_t prefix_first(const PrefixPieces& f, int hkv, int b, int kvh) {
  return (static_cast<int64_t>(b / (2 * f.tq)) * hkv + kvh) * f.S;
}
__device__ __forceinline__ int prefix_row(const PrefixPieces& f, int g, int b, int j) {
  return ((b / f.tq) & 1) * 128 + (b % f.tq) * g + j;
}

// Four outputs of one query head.
template <typename E, int D>
__device__ __forceinline__ void store4(const DecodeParams& p, int b, int head, int d4, float den, float4 num) {
  const float inv = den == 0.f ? 0.f : __frcp_rn(den);
  E* o = static_cast<E*>(p.out) + (static_cast<int64_t>(b) * p.hq + head) * D + d4 * 4;
  uint2 w;
  w.x = Elem<E>::pack(num.x * inv, num.y * inv);
  w.y = Elem<E>::pack(num.z * inv, num.w * inv);
  *reinterpret_cast<uint2*>(o) = w;
}

// A CTA's share of the units (an item's tiles, and item_tiles for its start and
// end): where it starts, how many it takes; x: the first one's place in its item.
struct Share {
  Shares all;
  long long count, pos;
  int b, hv, x;
};

// Taken by one whole warp.
template <class P>
__device__ __forceinline__ Share find_share(const P& p, int cta, int n_ctas) {
  const int lane = threadIdx.x & 31;
  const int hv = p.hkv * p.nrb;
  const long long pre = P::kPrefix ? static_cast<long long>(p.pre_items) * (p.pre_tiles + p.item_tiles) : 0;
  auto cost = [&](int b) {
    return b < p.B ? tiles_of(p, clamped_len(p.lens, b, p.len_limit)) + p.item_tiles : 0;
  };
  Share s;
  if (p.B <= 32 && p.n_units32) {
    // Up to 32 sequences and 2^31 units: one scan, and little code (a launch
    // fetches it from the L2 cache at first use, which is most of the time
    // that a short call takes here).
    const uint32_t c = cost(lane);
    uint32_t sum = c;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += t;
    }
    const uint32_t ahead = static_cast<uint32_t>(pre);  // prefix items come first, as sequence -1
    const uint32_t total = __shfl_sync(0xffffffffu, sum, 31) * hv + ahead;
    const uint32_t each = (total + n_ctas - 1) / n_ctas;
    const uint32_t pos = min(total, cta * each);
    s.all.total = total;
    s.all.each = each;
    s.pos = pos;
    s.count = min(total, pos + each) - pos;
    uint32_t per = p.pre_tiles + p.item_tiles, in = pos;
    s.b = -1;
    if (!P::kPrefix || pos >= ahead) {
      const unsigned past = __ballot_sync(0xffffffffu, sum * hv > pos - ahead);
      const int l = past ? __ffs(past) - 1 : 0;
      per = max(1u, __shfl_sync(0xffffffffu, c, l));
      in = pos - ahead - (__shfl_sync(0xffffffffu, sum, l) - per) * hv;
      s.b = l;
    }
    s.hv = in / per;
    s.x = in - s.hv * per;
    return s;
  }
  long long total = 0;
#pragma unroll 1
  for (int b = lane; b < p.B; b += 32) total += cost(b);
#pragma unroll 1
  for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
  s.all.set(total * hv + pre, n_ctas, 1);
  s.pos = s.all.begin(cta);
  s.count = s.all.begin(cta + 1) - s.pos;
  s.b = -1;
  s.hv = s.x = 0;
  if (s.count == 0) return s;
  long long before = 0;
  int per = p.pre_tiles + p.item_tiles;
  if (!P::kPrefix || s.pos >= pre) {  // (prefix items come first, as sequence -1)
    before = pre;
#pragma unroll 1
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int c = cost(b0 + lane);
      long long sum = static_cast<long long>(c) * hv;
#pragma unroll 1
      for (int off = 1; off < 32; off <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += t;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + sum > s.pos);
      if (past) {
        const int l = __ffs(past) - 1;
        per = __shfl_sync(0xffffffffu, c, l);
        before += __shfl_sync(0xffffffffu, sum, l) - static_cast<long long>(per) * hv;
        s.b = b0 + l;
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  s.hv = static_cast<int>(quotient(s.pos - before, per));
  s.x = static_cast<int>(s.pos - before - static_cast<long long>(s.hv) * per);
  return s;
}

// An item as the share walks over it.
struct Item {
  const int32_t* table;
  int len, tiles, kvh, head0, rows, first;  // first: the prefix's first sequence
  int units, x0, x1;                        // of the share that the item takes; tiles in it
};
template <class P>
__device__ __forceinline__ Item item_of(const P& p, const Share& s) {
  Item i;
  if (P::kPrefix && s.b < 0) {
    const int blocks = p.pre_items / p.hkv;
    i.kvh = s.hv / blocks;
    i.first = (s.hv - i.kvh * blocks) * p.pre_seqs;
    i.len = p.pre_len;
    i.tiles = p.pre_tiles;
    i.table = p.pre_table;
    i.head0 = i.kvh * p.g;
    i.rows = min(p.pre_seqs, p.B - i.first) * p.g;
  } else {
    i.len = clamped_len(p.lens, s.b, p.len_limit);
    i.tiles = tiles_of(p, i.len);
    i.table = p.table + s.b * p.table_stride;
    i.kvh = s.hv / p.nrb;
    const int rb = s.hv - i.kvh * p.nrb;
    i.head0 = i.kvh * p.g + rb * 16;
    i.rows = min(16, p.g - rb * 16);
    i.first = 0;
  }
  i.units = static_cast<int>(min(static_cast<long long>(i.tiles + p.item_tiles - s.x), s.count));
  i.x0 = max(0, s.x - p.item_tiles);
  i.x1 = max(0, s.x + i.units - p.item_tiles);
  return i;
}
// Behind n units of the item at hand.
template <class P>
__device__ __forceinline__ void advance(const P& p, Share& s, int n) {
  s.pos += n;
  s.count -= n;
  s.x = 0;
  if (++s.hv == (P::kPrefix && s.b < 0 ? p.pre_items : p.hkv * p.nrb)) {
    s.hv = 0;
    ++s.b;
  }
}
// First row of an item's whole result (see Params::part).
__device__ __forceinline__ int64_t whole_row(const DecodeParams& p, int b, int hv) {
  const int64_t cut = 2 * static_cast<int64_t>(p.n_ctas) * p.rows;
  if (b < 0) return cut + static_cast<int64_t>(hv) * 16;
  return cut + static_cast<int64_t>(p.pre_items) * 16 +
         (static_cast<int64_t>(b) * p.hkv * p.nrb + hv) * min(16, p.g);
}


// Joins an item's pieces, R query heads a block: those that the CTAs of the
// decode kernel left, and the shared prefix's behind them. The pieces are
// dealt to groups of threads (several loads of each in flight), whose results
// are joined in order. kMeans: a piece is the mean of its values (which may be as
// large as fp32 goes), not their sum, and counts by its weights' sum; no call has a
// prefix then.
constexpr int kJoinThreads = 256;

template <typename E, int D, int R, bool kMeans>
__global__ void __launch_bounds__(kJoinThreads)
    paged_join_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int kCells = R * (D / 4), kGroups = kJoinThreads / kCells;
  __shared__ float4 s_num[kGroups][kCells];
  __shared__ float2 s_ml[kGroups][kCells];
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int4 raw = __ldcg(reinterpret_cast<const int4*>(p.desc + blockIdx.x));
  const Desc d{raw.x, raw.y, raw.z, raw.w};
  const int kvh = d.hv / p.nrb, rb = d.hv - kvh * p.nrb;
  const int rows = min(16, p.g - rb * 16);
  if (d.pieces == 0 || static_cast<int>(blockIdx.y) * R >= rows) return;
  const int cell = threadIdx.x % kCells, group = threadIdx.x / kCells;
  const int row = blockIdx.y * R + cell % R, d4 = cell / R;
  // A streamed prefix's pieces are described as an item's are.
  Desc f{0, 0, 0, 0};
  int f_row = 0;
  if (!kMeans && p.pre_items) {
    const int pid = kvh * (p.pre_items / p.hkv) + d.b / p.pre_seqs;
    const int4 t = __ldcg(reinterpret_cast<const int4*>(p.desc + gridDim.x + pid));
    f = Desc{t.x, t.y, t.z, t.w};
    f_row = d.b % p.pre_seqs * p.g + row;
  }
  const int own = d.pieces, all = kMeans ? own : own + p.prefix.S + f.pieces;
  // Piece 0 lies in its CTA's second place, piece i > 0 in CTA + i's first; a
  // whole result in the item's own.
  auto row_of = [&](const Desc& e, int i) {
    return !kMeans && e.cta < 0 ? whole_row(p, e.b, e.hv)
                     : (2 * (static_cast<int64_t>(e.cta) + i) + (i == 0 ? 1 : 0)) * p.rows;
  };
  const int64_t pre = !kMeans && p.prefix.S ? prefix_first(p.prefix, p.hkv, d.b, kvh) : 0;
  const int pre_row = !kMeans && p.prefix.S ? prefix_row(p.prefix, p.g, d.b, rb * 16 + row) : 0;
  float m = -INFINITY, l = 0.f;
  float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
  if (row < rows) {
    constexpr int kBatch = 4;
    for (int i0 = group; i0 < all; i0 += kBatch * kGroups) {
      float pm[kBatch], pl[kBatch];
      float4 v[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = i0 + u * kGroups;
        pm[u] = -INFINITY;
        pl[u] = 0.f;
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < own || (!kMeans && i < all && p.pre_items)) {
          const int64_t at = i < own ? row_of(d, i) + row : row_of(f, i - own) + f_row;
          pm[u] = __ldcg(p.m + at);
          pl[u] = __ldcg(p.l + at);
          v[u] = __ldcg(reinterpret_cast<const float4*>(p.part + at * D) + d4);
        } else if (!kMeans && i < all) {
          const int64_t s = pre + i - own;
          pm[u] = __ldcg(p.prefix.ml + s * 512 + pre_row);
          pl[u] = __ldcg(p.prefix.ml + s * 512 + 256 + pre_row);
          v[u] = __ldcg(reinterpret_cast<const float4*>(p.prefix.o) + (s * (D / 4) + d4) * 256 + pre_row);
        }
      }
      float mx = m;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) mx = fmaxf(mx, pm[u]);
      const float mu = mx == -INFINITY ? 0.f : mx;
      float f = exp2_approx(m - mu);
      l *= f;
      if constexpr (kMeans) {
        f = l;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          pl[u] *= exp2_approx(pm[u] - mu);
          l += pl[u];
        }
        const float per = l == 0.f ? 0.f : __fdividef(1.f, l);
        f *= per;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) pl[u] *= per;
      }
      num.x *= f; num.y *= f; num.z *= f; num.w *= f;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if constexpr (kMeans) {
          f = pl[u];
        } else {
          f = exp2_approx(pm[u] - mu);
          l = fmaf(pl[u], f, l);
        }
        num.x = fmaf(v[u].x, f, num.x);
        num.y = fmaf(v[u].y, f, num.y);
        num.z = fmaf(v[u].z, f, num.z);
        num.w = fmaf(v[u].w, f, num.w);
      }
      m = mx;
    }
  }
  if (kGroups > 1) {
    s_num[group][cell] = num;
    s_ml[group][cell] = make_float2(m, l);
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) m = fmaxf(m, s_ml[k][cell].x);
    const float mu = m == -INFINITY ? 0.f : m;
    l = 0.f;
    num = make_float4(0.f, 0.f, 0.f, 0.f);
    float per = 0.f;
    if constexpr (kMeans) {
#pragma unroll
      for (int k = 0; k < kGroups; ++k) l = fmaf(s_ml[k][cell].y, exp2_approx(s_ml[k][cell].x - mu), l);
      per = l == 0.f ? 0.f : __fdividef(1.f, l);
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      float f = exp2_approx(s_ml[k][cell].x - mu);
      const float4 v = s_num[k][cell];
      if constexpr (kMeans)
        f *= s_ml[k][cell].y * per;
      else
        l = fmaf(s_ml[k][cell].y, f, l);
      num.x = fmaf(v.x, f, num.x);
      num.y = fmaf(v.y, f, num.y);
      num.z = fmaf(v.z, f, num.z);
      num.w = fmaf(v.w, f, num.w);
    }
  }
  if (row < rows) store4<E, D>(p, d.b, kvh * p.g + rb * 16 + row, d4, kMeans ? 1.f : l, num);
}

// Launches it behind the first kernel (cfg: that one's stream and attributes).
template <typename E, int D, bool kMeans = false>
cudaError_t launch_join(const DecodeParams& p, cudaLaunchConfig_t cfg) {
  // Query heads a join block takes: few, so that the pieces of a small batch
  // spread over many threads, but one where there is one.
  const int rows = p.g < 16 ? p.g : 16, per = rows == 1 ? 1 : 4;
  const int64_t items = !kMeans && (p.prefix.S || p.pre_items) ? static_cast<int64_t>(p.B) * p.hkv * p.nrb : p.n_ctas;
  if (items > 0x7fffffff) return cudaErrorInvalidValue;
  cfg.gridDim = dim3(static_cast<unsigned>(items), (rows + per - 1) / per);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  return per == 1 ? cudaLaunchKernelEx(&cfg, paged_join_kernel<E, D, 1, kMeans>, p)
                  : cudaLaunchKernelEx(&cfg, paged_join_kernel<E, D, 4, kMeans>, p);
}

}  // namespace
}  // namespace dqg
