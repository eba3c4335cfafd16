// Attention of whole prompts (or chunks of them) over a paged cache, and of a
// batch's queries over a prefix that all of its sequences share. No reference
// counterpart (the reference models the cache's bytes,
// dequant/byte_model.py:214-219).
//
//   o[t, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[t, h] . k_j - m)
//
// over the keys that token t sees: of sequence b with q_len new tokens at the
// end of kv_len cached ones, token i sees keys j < kv_len - q_len + i + 1
// (all kv_len when not causal); zero where it sees none.
//
// Rows are packed: with g query heads per KV head a 128-row tile holds
// floor(128 / g) tokens times g heads, so that every row of the products uses
// the same keys, whatever g is. An item is a pair of such tiles (256 rows) of
// one sequence and KV head; its work is counted in blocks of 128 keys, and all
// blocks of the call are cut into equal shares, one per SM, whatever the
// lengths and masks are. An item that lies in one share is finished by its
// CTA; one that is cut leaves its pieces (max, sum, O) in the workspace, and a
// second kernel joins them in order (no atomics, the same bits every time).
//
// The products run over whole blocks of keys for a whole tile, with weights of
// zero where a row sees nothing. A zero weight times an infinity would not be
// zero, so the values that some row of the pair does not see are looked at first,
// by two warps of their own beside the softmax: non-finite ones become zeros in
// shared memory (finite ones cost one fused multiply-add each), and rows that do
// see one take it from memory when the segment ends.
//
// One CTA per SM: one warp copies queries and page rows (tensor-map
// boxes, 128-byte swizzle, a ring of key and value blocks), one thread issues
// the products on the tensor cores (tcgen05: S = Q K^T from shared memory,
// O += P V with P in tensor memory), and each tile has four softmax warps, one
// thread a row. Tensor memory holds both tiles' S (fp32, 128 columns; with D =
// 128 P takes the place of S as it is formed) and O (fp32, D columns), so one tile's
// softmax runs while the other's products do. O stays in tensor memory over
// all blocks: the maximum that weights refer to is moved, and O rescaled, only
// when it grows by more than 2^8, which bounds the weights; the sums are
// fp32 and the division by them comes at the end. P is rounded to the values'
// 16-bit type for the second product (the tensor cores take both operands in
// one type); the sum is taken before the rounding.
//
// Measured (B200, a stream of calls whose inputs alternate between three sets):
// bf16, causal, 8192 tokens, 64 query and 8 KV heads of 128: 1005 us, 1.09
// PFLOP/s, 0.64 of a cuBLAS product's burst rate and 0.78 of its sustained one (the
// power cap holds the clock at 1.55 GHz; one launch alone, at 1.62, takes 887);
// fp16, 2048 tokens, 32 heads: 60 us (54 where the inputs stay in the L2 cache).
// What bounds it: a block pair (256 rows, 128 keys)
// takes 3220 cycles where its products take 2048 on the tensor cores and its
// exponentials 2048 on their unit. A tile's chain is its softmax, 1980 cycles
// (490 until its scores are read, 1420 for the weights at 11 cycles each where
// the unit needs 8, 70 to hand over), and then 1240 until its next scores are
// there (products of the late weights and of the next block, 768, and the
// signals between the warps); the other tile runs between, but not for free. An
// item's start and end cost about 3 us more. Tried and slower (8192 tokens, 989
// us on that GPU): every fourth weight by a polynomial on the fp32 pipe (1062: a lone
// warp is bound by issue, not by the unit), weights formed before the block's
// maximum is known (1012), two threads a row (1166), blocks of 64 keys with the
// scores one block ahead (1114: a product of 64 columns reads its operands at
// 2/3 of the rate, and its one issuing thread becomes the bound), a product
// warp for each tile (1182). With D = 64 the products are half as long and P has
// columns of its own, so the softmax alone bounds it (in a long prompt the
// exponential unit is busy 0.74 of the time, the tensor cores 0.37): 13 packed
// prompts, 6858 tokens, 32 and 8 heads: 107 us, 103 on warm inputs (115 with P in
// the place of S).
#include <cstdint>

#include "paged.cuh"

namespace dqg {
namespace {

constexpr int kBlock = 128;         // keys a block; rows a tile
constexpr int kThreads = 384;       // 2 x 4 softmax warps; products, copies, 2 value warps
constexpr int kMmaWarp = 8, kCopyWarp = 9, kValueWarp = 10, kValueWarps = 2;
// Weights are relative to a reference kHeadroom below a maximum that the true one
// exceeds by kMaxGrowth at most (log2 units): 2^15 at most, so that of fp16's
// range (2^-24 to 2^16) what lies above 1 is used too, and what a weight loses at
// the lower end is below 2^-32 of the largest one.
constexpr float kMaxGrowth = 8.f, kHeadroom = 7.f;
constexpr int kEarly = 96;          // keys whose weights are handed over first
// An item's start and end, in keys' time: 8192 tokens, 64/8 heads of 128, 1061 us
// with 128, 991 with 256, 981 with 512; 2048 tokens, 32 heads of 128, 57.1, 54.5,
// 55.8; 13 packed prompts, 32/8 heads of 64, 130, 103, 109; 8192 tokens of them 386,
// 364, 382.
constexpr int kItemKeys = 2 * kBlock;
constexpr int kSegs = 4;            // segments described ahead

struct Desc {  // a cut item, by the CTA that holds its first piece
  int tok0, ntok, kvh, pieces;
};

struct Params {
  const void* v;  // the pool of value pages
  const int32_t* table;
  const int32_t* q_starts;
  const int32_t* lens;
  void* out;
  float4* part;   // [slot][D / 4][256]
  float* ml;      // [slot][2][256]
  Desc* desc;     // [CTA]
  int64_t table_stride, n_pages, page_stride, head_stride, row_stride;
  int B, T, hq, hkv, g, tq, page_shift, len_limit, box_rows;
  bool causal;
  float scale_log2;
  uint32_t g_magic;                   // ceil(2^32 / g), 0 for g = 1
  bool n_units32;                     // the units of any lengths fit 31 bits
  int prefix_len, splits, n_pieces;   // a shared prefix: splits > 0
};

// ------------------------------------------------------------ tensor cores
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead_bytes, uint32_t stride_bytes) {
  // 128-byte swizzle; `stride` between groups of eight 128-byte rows, `lead`
  // between 64-value blocks of an operand whose contiguous dimension is not
  // the summed one.
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | static_cast<uint64_t>(lead_bytes >> 4) << 16 |
         static_cast<uint64_t>(stride_bytes >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
// fp32 accumulation of 16-bit operands; m = 128. b_rows: B's contiguous
// dimension is n (the values), not the summed one.
__device__ __forceinline__ constexpr uint32_t instr_desc(uint32_t format, uint32_t n, bool b_rows) {
  return 1u << 4 | format << 7 | format << 10 | (b_rows ? 1u : 0u) << 16 | (n >> 3) << 17 | (128u >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
      : "memory");
}
// Arrive on `bar` when every product this thread has issued is complete.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this thread's row of tensor memory.
#define DQG_R8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
#define DQG_W8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define DQG_U8(a, i) "+r"(a[i]), "+r"(a[i + 1]), "+r"(a[i + 2]), "+r"(a[i + 3]), "+r"(a[i + 4]), "+r"(a[i + 5]), "+r"(a[i + 6]), "+r"(a[i + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : DQG_W8(r, 0), DQG_W8(r, 8), DQG_W8(r, 16), DQG_W8(r, 24)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::DQG_R8(r, 0),
      DQG_R8(r, 8), DQG_R8(r, 16), DQG_R8(r, 24), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::DQG_R8(r, 0),
      DQG_R8(r, 8), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Uses of r stay behind the wait that precedes this.
__device__ __forceinline__ void hold32(uint32_t* r) {
  asm volatile("" : DQG_U8(r, 0), DQG_U8(r, 8), DQG_U8(r, 16), DQG_U8(r, 24));
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// ---------------------------------------------------------------- schedule
struct Seq {  // one sequence's rows and keys
  int q0, ql, kv, pairs;
};
__device__ __forceinline__ int blocks_of(int keys) { return keys > 0 ? (keys + kBlock - 1) / kBlock : 1; }

__device__ __forceinline__ Seq load_seq(const Params& p, int b) {
  Seq s;
  if (p.splits) {
    s.q0 = 0;
    s.ql = p.T;
    s.kv = p.prefix_len;
  } else {
    s.q0 = __ldg(p.q_starts + b);
    s.ql = __ldg(p.q_starts + b + 1) - s.q0;
    s.kv = clamped_len(p.lens, b, p.len_limit);
    // Starts out of order or range: no rows.
    if (s.q0 < 0 || s.ql < 0 || s.q0 > p.T || s.ql > p.T - s.q0) {
      s.ql = 0;
      atomicOr(&g_status, kStatusBadIndex);
    }
  }
  s.pairs = (s.ql + 2 * p.tq - 1) / (2 * p.tq);
  return s;
}

// Keys that a tile whose last token is i sees: its block count follows.
__device__ __forceinline__ int limit_of(const Params& p, const Seq& s, int i) {
  if (!p.causal) return s.kv;
  const int lim = s.kv - s.ql + i + 1;
  return lim < 0 ? 0 : lim;
}

// The cost of an item: the keys that its last token sees, and kItemKeys for its
// start and end. (Keys, not blocks: their sum over a causal sequence's pairs is
// a plain quadratic, which every CTA evaluates to find its share.)
// Cost of a sequence's first n pairs, for one KV head.
__device__ __forceinline__ long long cost_before(const Params& p, const Seq& s, int n) {
  const long long start = static_cast<long long>(n) * kItemKeys;
  if (n <= 0) return 0;
  if (!p.causal) return start + static_cast<long long>(n) * s.kv;
  const int tokens = 2 * p.tq, off = s.kv - s.ql;
  const int full = n < s.pairs ? n : s.pairs - 1;  // the last pair ends at kv
  const int none = off < 0 ? min(full, -off / tokens) : 0;  // pairs that see no key
  const long long k = full - none;
  const long long first = off + static_cast<long long>(none) * tokens;
  return start + k * first + k * (k + 1) / 2 * tokens + (n == s.pairs ? s.kv : 0);
}
// The block where a cut `unit` units into an item falls.
__device__ __forceinline__ int cut_block(int unit) {
  return unit < kItemKeys ? 0 : (unit - kItemKeys + kBlock / 2) / kBlock;
}

struct Share {  // a CTA's part of the units; x: the first one's place in its item
  Shares all;
  long long count, pos;
  int b, kvh, pair, x;
};

// Taken by one whole warp; *s: the sequence where the share starts.
__device__ __forceinline__ Share find_share(const Params& p, int cta, int n_ctas, Seq* s) {
  const int lane = threadIdx.x & 31;
  Share r;
  r.b = r.kvh = r.pair = r.x = 0;
  long long in;
  if (p.B <= 32 && p.n_units32) {
    // Up to 32 sequences and 2^31 units: one scan, and little code (a launch
    // fetches it from the L2 cache at first use, which is most of the time
    // that a short call takes here).
    Seq mine = {0, 0, 0, 0};
    if (lane < p.B) mine = load_seq(p, lane);
    const uint32_t c = static_cast<uint32_t>(cost_before(p, mine, mine.pairs));
    uint32_t sum = c;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += t;
    }
    const uint32_t total = __shfl_sync(0xffffffffu, sum, 31) * p.hkv;
    const uint32_t each = max((total + n_ctas - 1) / n_ctas, static_cast<uint32_t>(kBlock));
    const uint32_t pos = min(total, cta * each);
    r.all.total = total;
    r.all.each = each;
    r.pos = pos;
    r.count = min(total, pos + each) - pos;
    const unsigned past = __ballot_sync(0xffffffffu, sum * p.hkv > pos);
    const int l = past ? __ffs(past) - 1 : 0;
    const uint32_t per = max(1u, __shfl_sync(0xffffffffu, c, l));
    const uint32_t rest = pos - (__shfl_sync(0xffffffffu, sum, l) - per) * p.hkv;
    r.b = l;
    r.kvh = rest / per;
    in = rest - r.kvh * per;
    s->q0 = __shfl_sync(0xffffffffu, mine.q0, l);
    s->ql = __shfl_sync(0xffffffffu, mine.ql, l);
    s->kv = __shfl_sync(0xffffffffu, mine.kv, l);
    s->pairs = __shfl_sync(0xffffffffu, mine.pairs, l);
    if (r.count == 0) return r;
  } else {
    long long total = 0;
#pragma unroll 1
    for (int b = lane; b < p.B; b += 32) {
      const Seq t = load_seq(p, b);
      total += cost_before(p, t, t.pairs);
    }
#pragma unroll 1
    for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    // Shares of a block at least, so that none inside an item comes to nothing.
    r.all.set(total * p.hkv, n_ctas, kBlock);
    r.pos = r.all.begin(cta);
    r.count = r.all.begin(cta + 1) - r.pos;
    if (r.count == 0) return r;
    long long before = 0, per = 1;
#pragma unroll 1
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int b = b0 + lane;
      long long mine = 0;
      if (b < p.B) {
        const Seq t = load_seq(p, b);
        mine = cost_before(p, t, t.pairs);
      }
      long long sum = mine * p.hkv;
#pragma unroll 1
      for (int off = 1; off < 32; off <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += t;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + sum > r.pos);
      if (past) {
        const int l = __ffs(past) - 1;
        per = __shfl_sync(0xffffffffu, mine, l);
        before += __shfl_sync(0xffffffffu, sum, l) - per * p.hkv;
        r.b = b0 + l;
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    in = r.pos - before;
    r.kvh = static_cast<int>(quotient(in, per));
    in -= r.kvh * per;
    *s = load_seq(p, r.b);
  }
  // The pair: 32 probes a round.
  int lo = 0, hi = s->pairs;
#pragma unroll 1
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int probe = min(lo + (lane + 1) * step, hi);
    const int f = __ffs(__ballot_sync(0xffffffffu, cost_before(p, *s, probe) > in)) - 1;
    hi = min(lo + (f + 1) * step, hi);
    lo = lo + f * step;
  }
  r.pair = lo;
  r.x = static_cast<int>(in - cost_before(p, *s, lo));
  return r;
}

// What a CTA does next: blocks [x0, x1) of one item. The copying warp walks
// the CTA's share and describes each segment to the other warps.
struct Segment {
  int kvh, tok0, ntok, x0, x1, slot;  // tok0, ntok: the pair's tokens, rows of q
  int n0, n1;                         // the tiles' blocks over the whole item; n1 = 0: no second tile
  int kv, lim0;                       // keys; keys that the first token sees (or below 0)
  int whole;                          // the item lies in this segment
  int pieces;                         // of the item, where this is the first of several
  int b;                              // sequence
  int from, check;                    // the value warps look at keys >= from, in blocks >= check
  int tainted;                        // such a key's values were not finite (set by the value warps)
};
// Blocks of a segment that tile t takes part in.
__device__ __forceinline__ int tile_count(const Segment& g, int t) {
  const int n = t ? g.n1 : g.n0;
  return max(0, min(g.x1, n) - g.x0);
}

struct Walk {
  Share r;
  Seq s;
  int piece;
  __device__ __forceinline__ void begin(const Params& p) {
    piece = blockIdx.x;
    if (p.splits)
      s = load_seq(p, 0);
    else
      r = find_share(p, blockIdx.x, gridDim.x, &s);
  }
  __device__ __forceinline__ void tiles(const Params& p, Segment& g, int pair) {
    const int first = pair * 2 * p.tq;  // the pair's first token in its sequence
    g.tok0 = s.q0 + first;
    g.ntok = min(2 * p.tq, s.ql - first);
    g.n0 = blocks_of(limit_of(p, s, first + min(p.tq, g.ntok) - 1));
    g.n1 = g.ntok > p.tq ? blocks_of(limit_of(p, s, first + g.ntok - 1)) : 0;
    g.kv = s.kv;
    g.lim0 = s.kv - s.ql + first + 1;
  }
  __device__ __forceinline__ bool next(const Params& p, Segment& g, int& b) {
    if (p.splits) {
      if (piece >= p.n_pieces) return false;
      const int item = piece / p.splits, sp = piece - item * p.splits;
      const int pair = item / p.hkv;
      b = 0;
      g.kvh = item - pair * p.hkv;
      tiles(p, g, pair);
      const int n = g.n0;  // both tiles see every key
      g.x0 = static_cast<int>(static_cast<long long>(sp) * n / p.splits);
      g.x1 = static_cast<int>(static_cast<long long>(sp + 1) * n / p.splits);
      g.whole = 0;
      g.pieces = 0;
      g.slot = piece;
      piece += gridDim.x;
      return true;
    }
    while (r.count > 0) {
      b = r.b;
      g.kvh = r.kvh;
      tiles(p, g, r.pair);
      const int n = max(g.n0, g.n1);
      const int seen = max(0, limit_of(p, s, g.tok0 - s.q0 + g.ntok - 1));
      const int cost = seen + kItemKeys;
      const int end = static_cast<int>(min(static_cast<long long>(cost), r.x + r.count));
      g.x0 = min(n, cut_block(r.x));
      g.x1 = end == cost ? n : min(n, cut_block(end));
      g.whole = g.x0 == 0 && g.x1 == n;
      g.slot = 2 * blockIdx.x + (g.x0 > 0 ? 0 : 1);
      g.pieces = 0;
      if (!g.whole && g.x0 == 0 && g.x1 > 0) {
        // The last piece lies with the holder of the item's last unit, unless
        // that one's cut falls behind the last block.
        const long long start = r.pos - r.x;
        const int last = r.all.holder(start + cost - 1);
        g.pieces = last - static_cast<int>(blockIdx.x) + 1 -
                   (cut_block(static_cast<int>(r.all.begin(last) - start)) >= n ? 1 : 0);
      }
      r.pos += end - r.x;
      r.count -= end - r.x;
      r.x = 0;
      if (r.count > 0 && ++r.pair == s.pairs) {
        r.pair = 0;
        if (++r.kvh == p.hkv) {
          r.kvh = 0;
          do {
            s = load_seq(p, ++r.b);
          } while (s.pairs == 0);  // a share never ends in sequences without rows
        }
      }
      if (g.x1 > g.x0) return true;
    }
    return false;
  }
};

// ------------------------------------------------------------------ kernel
template <int D>
struct Layout {
  static constexpr int kStages = D == 128 ? 4 : 8;     // key or value blocks in flight
  static constexpr int kSlot = kBlock * D * 2;
  // With D = 64 tensor memory has room for P beside S: the next block's scores
  // are formed while a block's weights still are.
  static constexpr bool kApart = D == 64;
  static constexpr int kTile = 128 * D * 2;            // a tile's queries
  static constexpr int kRing = 2 * kTile;              // offset of the ring
  static constexpr int kStore = kRing + kStages * kSlot;  // 4 KB a softmax warp, for its stores
  static constexpr int kBars = kStore + 8 * 4096;
  static constexpr int kBarBytes = (4 * kStages + 11 + 2 * kSegs) * 8 + kSegs * static_cast<int>(sizeof(Segment)) + 8;
  static constexpr int kSmem = 1024 + kBars + kBarBytes;
};

// Zeros in place of the non-finite values in rows [r0, r1) of a block in shared
// memory (128 rows in halves of 64 values); whether one of the first `rows` rows
// held one. r0 is a multiple of 4. Taken by the value warps, `part` of them each.
template <typename E, int D>
__device__ __forceinline__ bool clean_values(uint8_t* v, int r0, int r1, int rows, int part) {
  const int lane = threadIdx.x & 31;
  uint32_t acc[4] = {0u, 0u, 0u, 0u};  // 0 x = 0 for every finite x, NaN otherwise
#pragma unroll 4
  for (int r = r0 + 4 * part; r < r1; r += 4 * kValueWarps) {
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
      const uint4 w = *reinterpret_cast<const uint4*>(v + h * (kBlock * 128) + r * 128 + lane * 16);
      acc[0] = Elem<E>::fma2(w.x, 0u, acc[0]);
      acc[1] = Elem<E>::fma2(w.y, 0u, acc[1]);
      acc[2] = Elem<E>::fma2(w.z, 0u, acc[2]);
      acc[3] = Elem<E>::fma2(w.w, 0u, acc[3]);
    }
  }
  if (!__any_sync(0xffffffffu, (acc[0] | acc[1] | acc[2] | acc[3]) != 0u)) return false;
  bool seen = false;
#pragma unroll 1
  for (int i = 0; i < D / 64 * kBlock; i += 4) {  // (rows of both halves)
    const int r = i % kBlock;
    if (r < r0 || r >= r1 || (r / 4) % kValueWarps != (r0 / 4 + part) % kValueWarps) continue;
    uint4* at = reinterpret_cast<uint4*>(v + i * 128 + lane * 16);
    uint4 w = *at;
    uint32_t* ww = reinterpret_cast<uint32_t*>(&w);
    bool any = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t bad = Elem<E>::non_finite(ww[e]);
      any |= bad != 0u;
      ww[e] &= ~bad;
    }
    if (any) {
      *at = w;
      seen |= r + (lane >> 3) < rows;
    }
  }
  return __any_sync(0xffffffffu, seen);
}

// Adds to this thread's row of tile `tile` the non-finite values, among the keys
// that it sees, which clean_values took out of a segment's products. (A key that
// a row sees has a positive weight, whatever a 16-bit type makes of it.) Taken by
// the tile's softmax warps; rare, and out of line, where it takes no registers
// from them.
template <typename E, int D>
__device__ __noinline__ void take_non_finite(const Params& p, const Segment& g, int tile, uint32_t tmem) {
  const uint32_t to = tmem + (((threadIdx.x >> 5) & 3) << 21) + 2 * kBlock + tile * D;
  const int token = tile * p.tq + (threadIdx.x & 127) / p.g;
  const int limit = p.causal ? min(g.lim0 + token, g.kv) : g.kv;
  const int from = max(g.from, g.x0 * kBlock), end = min(g.kv, (g.x0 + tile_count(g, tile)) * kBlock);
  const int32_t* table = p.table + g.b * p.table_stride;
  const E* pool = static_cast<const E*>(p.v) + g.kvh * p.head_stride;
  const int in_page = (1 << p.page_shift) - 1;
#pragma unroll 1
  for (int q = 0; q < D / 32; ++q) {
    uint32_t o[32];
    tmem_ld32(to + 32 * q, o);
    tmem_wait_ld();
    hold32(o);
#pragma unroll 1
    for (int t = from; t < end; ++t) {
      const int page = __ldg(table + (t >> p.page_shift));
      if (page < 0 || page >= p.n_pages) continue;
      const uint4* row =
          reinterpret_cast<const uint4*>(pool + page * p.page_stride + (t & in_page) * p.row_stride + 32 * q);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 w = row[i];
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bad = Elem<E>::non_finite(ww[e]);
          if (bad != 0u && t < limit) {
            const float2 x = Elem<E>::unpack(ww[e] & bad);
            o[8 * i + 2 * e] = __float_as_uint(__uint_as_float(o[8 * i + 2 * e]) + x.x);
            o[8 * i + 2 * e + 1] = __float_as_uint(__uint_as_float(o[8 * i + 2 * e + 1]) + x.y);
          }
        }
      }
    }
    __syncwarp();
    tmem_st32(to + 32 * q, o);
  }
  tmem_wait_st();
}

template <typename E, int D>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap qmap,
                  const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using L = Layout<D>;
  constexpr int kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* full = bars;                 // ring slots
  uint64_t* empty = full + kStages;
  uint64_t* q_full = empty + kStages;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;        // [2], one a tile
  uint64_t* p_half = s_full + 2;
  uint64_t* p_full = p_half + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* seg_full = o_full + 2;       // [kSegs]
  uint64_t* seg_empty = seg_full + kSegs;
  uint64_t* drained = seg_empty + kSegs;
  uint64_t* asked = drained + 1;         // [kStages], in the order of the checked blocks:
  uint64_t* checked = asked + kStages;   // values on their way; values checked
  Segment* segs = reinterpret_cast<Segment*>(checked + kStages);  // [kSegs]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(segs + kSegs);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sbase = smem_u32(smem);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
      mbar_init(asked + i, 1);
      mbar_init(checked + i, kValueWarps);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full + t, 1);
      mbar_init(p_half + t, 128);
      mbar_init(p_full + t, 128);
      mbar_init(o_full + t, 1);
    }
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(seg_full + i, 1);
      mbar_init(seg_empty + i, 9 + kValueWarps);
    }
    mbar_init(drained, 1);
    fence_mbar_init();
    tma_prefetch_map(&qmap);
    tma_prefetch_map(&kmap);
    tma_prefetch_map(&vmap);
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // Rows that no (token, head) fills stay zero for the whole kernel.
  const int used = p.tq * p.g;
  if (used < 128) {
    for (int i = threadIdx.x; i < 2 * (D / 64) * (128 - used) * 8; i += kThreads) {
      const int ch = i & 7, rest = i >> 3;
      const int r = used + rest % (128 - used), blk = rest / (128 - used);
      *reinterpret_cast<uint4*>(smem + blk * (128 * 128) + r * 128 + ch * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_async_shared();
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const uint32_t tmem = *tmem_slot;
  // Registers: a softmax thread holds a row of 128 scores. 384 x 168 at
  // launch = 256 x 216 + 128 x 72.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == kCopyWarp) {
      // ---- copies: queries per segment, then key and value blocks in turn.
      Walk walk;
      walk.begin(p);
      Segment g;
      const int per = p.box_rows, boxes = kBlock / per * (D / 64);
      const int half = lane % (D / 64), sub = lane / (D / 64);
      int seg = 0, pos = 0, checks = 0;
      bool ok = true;
      while (ok) {
        int b = 0;
        const bool more = walk.next(p, g, b);
        const int sg = seg % kSegs;
        if (seg >= kSegs && !warp_wait(seg_empty + sg, ((seg / kSegs) & 1) ^ 1)) break;
        g.from = max(0, p.causal ? g.lim0 : g.kv) & ~3;
        g.check = max(g.x0, g.from / kBlock);
        if (lane == 0) {
          if (!more) g.x0 = g.x1 = 0;  // the end
          g.b = b;
          g.tainted = 0;
          segs[sg] = g;
          mbar_arrive(seg_full + sg);
        }
        if (!more) break;
        if (seg > 0 && !warp_wait(q_empty, (seg - 1) & 1)) break;
        const int tiles = g.n1 > 0 ? 2 : 1;
        if (lane == 0) mbar_arrive_expect_tx(q_full, tiles * used * D * 2);
        __syncwarp();
        if (lane < tiles * (D / 64)) {
          const int t = lane / (D / 64), h = lane % (D / 64);
          tma_load_4d(sbase + t * L::kTile + h * (128 * 128), &qmap, q_full, h * 64, 0, g.kvh, g.tok0 + t * p.tq);
        }
        ++seg;
        const int32_t* row = p.table + b * p.table_stride;
        if (!p.splits && lane == 0 && __ldg(p.lens + b) != g.kv) atomicOr(&g_status, kStatusBadIndex);
        for (int x = g.x0; x < g.x1 && ok; ++x) {
          const int t = x * kBlock + sub * per;
          int page = static_cast<int>(p.n_pages);  // no such page: zeros
          if (lane < boxes && t < g.kv) {
            page = __ldg(row + (t >> p.page_shift));
            if (page < 0 || page >= p.n_pages) {
              page = static_cast<int>(p.n_pages);
              atomicOr(&g_status, kStatusBadIndex);
            }
          }
          const int in_page = t & ((1 << p.page_shift) - 1);
          for (int w = 0; w < 2; ++w, ++pos) {
            const int st = pos % kStages;
            if (pos >= kStages && !warp_wait(empty + st, ((pos / kStages) & 1) ^ 1)) {
              ok = false;
              break;
            }
            if (lane == 0) mbar_arrive_expect_tx(full + st, L::kSlot);
            __syncwarp();
            if (lane < boxes)
              tma_load_4d(sbase + L::kRing + st * L::kSlot + half * (kBlock * 128) + sub * per * 128,
                          w ? &vmap : &kmap, full + st, half * 64, in_page, g.kvh, page);
          }
          if (ok && x >= g.check) {
            if (lane == 0) mbar_arrive(asked + checks % kStages);
            ++checks;
          }
        }
      }
      // Copies still in flight land before the CTA's memory goes (bounded).
      if (seg > 0) warp_wait(q_full, (seg - 1) & 1);
      for (int i = pos < kStages ? 0 : pos - kStages; i < pos; ++i)
        if (!warp_wait(full + i % kStages, (i / kStages) & 1)) break;
    } else if (warp == kMmaWarp) {
      // ---- products: one elected thread waits for what they need and issues them.
      constexpr uint32_t kIdS = instr_desc(Elem<E>::kFormat, kBlock, false);
      constexpr uint32_t kIdO = instr_desc(Elem<E>::kFormat, D, true);
      if (elect_one()) {
        const uint64_t q_desc = smem_desc(sbase, 16, 1024);
        const uint64_t k_desc = smem_desc(sbase + L::kRing, 16, 1024);
        const uint64_t v_desc = smem_desc(sbase + L::kRing, kBlock * 128, 1024);
        auto issue_s = [&](int t, int slot) {
          const uint64_t a = q_desc + t * (L::kTile >> 4), b = k_desc + slot * (L::kSlot >> 4);
    #pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = ((k / 4) * (128 * 128) + (k % 4) * 32) >> 4;
            mma_ss(tmem + t * kBlock, a + off, b + off, kIdS, k > 0);
          }
          mma_commit(s_full + t);
        };
        const uint32_t weights_at = L::kApart ? tmem + 2 * kBlock + 2 * D : tmem;
        constexpr uint32_t weights_step = L::kApart ? kBlock / 2 : kBlock;
        auto issue_o = [&](int t, int slot, bool late, bool add) {
          const uint64_t b = v_desc + slot * (L::kSlot >> 4);
    #pragma unroll
          for (int k = 0; k < kBlock / 16; ++k) {
            if ((k < kEarly / 16) != late)
              mma_ts(tmem + 2 * kBlock + t * D, weights_at + t * weights_step + k * 8, b + (k * 16 * 128 >> 4), kIdO,
                     add || k > 0);
          }
        };
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          const bool ok = mbar_wait(bar, parity);
          fence_after_sync();
          return ok;
        };
        int seg = 0, slot = 0;
        uint32_t ring = 0, weights = 0;  // parities: the ring's, the two tiles' weights
        auto advance = [&] {
          if (++slot == kStages) {
            slot = 0;
            ring ^= 1;
          }
        };
        bool ok = true;
        while (ok) {
          const int sg = seg % kSegs;
          if (!mbar_wait(seg_full + sg, (seg / kSegs) & 1)) break;
          const int c0 = tile_count(segs[sg], 0), c1 = tile_count(segs[sg], 1);
          const int n = segs[sg].x1 - segs[sg].x0;
          if (n == 0) break;
          mbar_arrive(seg_empty + sg);
          ok = wait(q_full, seg & 1) && wait(full + slot, ring);
          ++seg;
          if (!ok) break;
          if (c0 > 0) issue_s(0, slot);
          if (c1 > 0) issue_s(1, slot);
          mma_commit(empty + slot);
          if (n == 1) mma_commit(q_empty);
          advance();
          for (int j = 0; j < n && ok; ++j) {
            const int vslot = slot;
            const bool more = j + 1 < n;
            ok = wait(full + vslot, ring);
            advance();
            const int kslot = slot;
            if (ok && more) {
              ok = wait(full + kslot, ring);
              advance();
            }
    #pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int c = t ? c1 : c0;
              if (!ok || j >= c) continue;
              ok = wait(p_half + t, weights >> t & 1);
              if (!ok) continue;
              // (Early weights also say that the block's scores have been read.)
              if (L::kApart && j + 1 < c) issue_s(t, kslot);
              issue_o(t, vslot, false, j > 0);
              ok = wait(p_full + t, weights >> t & 1);
              weights ^= 1u << t;
              if (!ok) continue;
              issue_o(t, vslot, true, true);
              if (!L::kApart && j + 1 < c) issue_s(t, kslot);
              else mma_commit(o_full + t);
            }
            mma_commit(empty + vslot);
            if (more) mma_commit(empty + kslot);
            if (j + 2 == n) mma_commit(q_empty);
          }
        }
        // Nothing of this CTA is in flight when it ends (bounded).
        mma_commit(drained);
        mbar_wait(drained, 0);
      }
      __syncwarp();
    } else {
      // ---- values that not every row sees. Blocks that need no look are not
      // waited for, so the copies say when one that does is on its way: the phase
      // of its ring slot is then the current one, and stays so until the products
      // have taken it, which these warps have to let them first. (For the same reason
      // no phase of `asked` or `checked` is ever overrun.)
      int seg = 0, base = 0, n = 0;
      bool ok = true;
      while (ok) {
        const int sg = seg % kSegs;
        if (!warp_wait(seg_full + sg, (seg / kSegs) & 1)) break;
        Segment& g = segs[sg];
        const int x0 = g.x0, x1 = g.x1, kv = g.kv;
        if (x1 == x0) break;
        ++seg;
        for (int x = g.check; x < x1; ++x, ++n) {
          const int pos = base + 2 * (x - x0) + 1;
          if (!warp_wait(asked + n % kStages, (n / kStages) & 1) ||
              !warp_wait(full + pos % kStages, (pos / kStages) & 1)) {
            ok = false;
            break;
          }
          // Rows of the last page behind the end hold anything, those of no page zeros.
          const int rows = kv - x * kBlock, end = ((rows - 1) | ((1 << p.page_shift) - 1)) + 1;
          if (clean_values<E, D>(smem + L::kRing + (pos % kStages) * L::kSlot, max(0, g.from - x * kBlock),
                                 min(kBlock, end), rows, warp - kValueWarp))
            g.tainted = 1;
          fence_async_shared();  // before the products read them
          __syncwarp();
          if (lane == 0) mbar_arrive(checked + n % kStages);
        }
        base += 2 * (x1 - x0);
        if (ok && lane == 0) mbar_arrive(seg_empty + sg);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---- softmax: one thread a row of tile t.
    const int t = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's 32 lanes
    const uint32_t ts = tmem + lanes + t * kBlock, to = tmem + lanes + 2 * kBlock + t * D;
    const uint32_t tp = L::kApart ? tmem + lanes + 2 * kBlock + 2 * D + t * (kBlock / 2) : ts;  // weights
    const int tok = t * p.tq + r / p.g;  // of the pair
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    int seg = 0, scores = 0, outs = 0, checks = 0;
    bool ok = true, cut_first = false;
    while (true) {
      const int sg = seg % kSegs;
      if (!warp_wait(seg_full + sg, (seg / kSegs) & 1)) break;
      const Segment& g = segs[sg];
      const int x0 = g.x0, kv = g.kv, n = tile_count(g, t), all = g.x1 - x0;
      if (all == 0) break;
      ++seg;
      const int limit = p.causal ? min(g.lim0 + tok, kv) : kv;
      // Keys that every row of the tile sees (rows past the end see no fewer).
      const int seen = p.causal ? g.lim0 + t * p.tq : kv;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j) {
        const int k0 = (x0 + j) * kBlock;
        if (!warp_wait(s_full + t, scores & 1)) {
          ok = false;
          break;
        }
        ++scores;
        fence_after_sync();
        uint32_t raw[128];
        float* s = reinterpret_cast<float*>(raw);
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(ts + 32 * q, raw + 32 * q);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q) hold32(raw + 32 * q);
        if (k0 + kBlock > seen) {
          const int left = limit - k0;
#pragma unroll
          for (int i = 0; i < kBlock; ++i) s[i] = i < left ? s[i] : -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < kBlock; i += 4)
#pragma unroll
          for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], s[i + q]);
        const float m_new = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), m);
        const bool grow = (m_new - m) * p.scale_log2 > kMaxGrowth;
        if (L::kApart && j > 0) {
          // The block before has to be in O, and its weights read, before
          // either changes (with P in the place of S its scores say so).
          if (!warp_wait(o_full + t, outs & 1)) {
            ok = false;
            break;
          }
          ++outs;
          fence_after_sync();
        }
        if (j == 0) {
          m = m_new;  // no O yet: the first product overwrites it
        } else if (__any_sync(0xffffffffu, grow)) {
          const float f = grow ? exp2_approx((m - m_new) * p.scale_log2) : 1.f;
#pragma unroll
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            tmem_ld32(to + 32 * q, o);
            tmem_wait_ld();
            hold32(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st32(to + 32 * q, o);
          }
          l *= f;
          if (grow) m = m_new;
        }
        const float ref = m == -INFINITY ? 0.f : fmaf(m, p.scale_log2, -kHeadroom);
        const float2 ref2 = make_float2(-ref, -ref);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // The products take the first kEarly weights while the rest is formed.
        auto weigh = [&](int from, uint32_t* w, int n) {
#pragma unroll
          for (int i = 0; i < n / 2; ++i) {
            float2 x = fma2(make_float2(s[from + 2 * i], s[from + 2 * i + 1]), scale2, ref2);
            x.x = exp2_approx(x.x);
            x.y = exp2_approx(x.y);
            sum[i & 1] = add2(sum[i & 1], x);
            w[i] = Elem<E>::pack(x.x, x.y);
          }
        };
        {
          uint32_t w[kEarly / 2];
          weigh(0, w, kEarly);
          tmem_st32(tp, w);
          tmem_st16(tp + 32, w + 32);
          if (x0 + j >= g.check) {
            const int c = checks + x0 + j - g.check;
            if (!warp_wait(checked + c % kStages, (c / kStages) & 1)) {
              ok = false;
              break;
            }
          }
          tmem_wait_st();
          fence_before_sync();
          mbar_arrive(p_half + t);
        }
        {
          uint32_t w[(kBlock - kEarly) / 2];
          weigh(kEarly, w, kBlock - kEarly);
          tmem_st16(tp + kEarly / 2, w);
          tmem_wait_st();
          fence_before_sync();
          mbar_arrive(p_full + t);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      checks += max(0, x0 + all - g.check);
      if (!ok) break;
      if (g.pieces && threadIdx.x == 0) p.desc[blockIdx.x] = Desc{g.tok0, g.ntok, g.kvh, g.pieces};
      cut_first |= g.pieces != 0;
      if (n > 0) {
        if (!warp_wait(o_full + t, outs & 1)) break;
        ++outs;
        fence_after_sync();
        if (g.tainted) take_non_finite<E, D>(p, g, t, tmem);
      }
      if ((t ? g.n1 : g.n0) > 0) {
        if (g.whole) {
          // 64 columns at a time through shared memory, so that a warp's
          // stores are whole 128-byte rows.
          const float inv = l == 0.f ? 0.f : __frcp_rn(l);
          uint8_t* st = smem + L::kStore + warp * 4096;
          E* out = static_cast<E*>(p.out) + static_cast<int64_t>(g.tok0) * p.hq * D + static_cast<int64_t>(g.kvh) * p.g * D;
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            uint32_t o[64];
            tmem_ld32(to + 64 * h, o);
            tmem_ld32(to + 64 * h + 32, o + 32);
            tmem_wait_ld();
            hold32(o);
            hold32(o + 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              uint4 w;
              uint32_t* ww = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                ww[e] = Elem<E>::pack(__uint_as_float(o[8 * i + 2 * e]) * inv,
                                      __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
              *reinterpret_cast<uint4*>(st + lane * 128 + ((i ^ (lane & 7)) << 4)) = w;
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int row = i * 4 + (lane >> 3), rr = (warp & 3) * 32 + row;
              const int tk = fast_div(rr, p.g_magic), head = rr - tk * p.g;
              if (rr < used && t * p.tq + tk < g.ntok)
                *reinterpret_cast<uint4*>(out + (static_cast<int64_t>(t * p.tq + tk) * p.hq + head) * D + 64 * h +
                                          (lane & 7) * 8) =
                    *reinterpret_cast<const uint4*>(st + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
            }
            __syncwarp();
          }
        } else {
          const int64_t slot = g.slot;
          p.ml[slot * 512 + t * 128 + r] = n > 0 && m != -INFINITY ? fmaf(m, p.scale_log2, -kHeadroom) : -INFINITY;
          p.ml[slot * 512 + 256 + t * 128 + r] = l;
#pragma unroll
          for (int q = 0; q < D / 32; ++q) {
            uint32_t o[32];
            if (n > 0) {
              tmem_ld32(to + 32 * q, o);
              tmem_wait_ld();
              hold32(o);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = 0u;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
              p.part[(slot * (D / 4) + q * 8 + i) * 256 + t * 128 + r] =
                  make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                              __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
          }
        }
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(seg_empty + sg);
    }
    if (threadIdx.x == 0 && !cut_first && !p.splits) p.desc[blockIdx.x] = Desc{0, 0, 0, 0};
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Joins the pieces of the item whose first piece CTA blockIdx.x holds: 32 rows
// a block, a lane a row, a warp eight columns.
template <typename E, int D>
__global__ void __launch_bounds__(32 * (D / 8)) prompt_join_kernel(const __grid_constant__ Params p) {
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  const int4 d = __ldcg(reinterpret_cast<const int4*>(p.desc + blockIdx.x));
  const int tok0 = d.x, ntok = d.y, kvh = d.z, pieces = d.w;
  if (pieces == 0) return;
  const int row = blockIdx.y * 32 + (threadIdx.x & 31), r = row & 127, d8 = threadIdx.x >> 5;
  const int tok = (row >> 7) * p.tq + r / p.g;
  if (r >= p.tq * p.g || tok >= ntok) return;
  constexpr int kBatch = 4;  // pieces whose loads are in flight together
  float m = -INFINITY, den = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < pieces; i0 += kBatch) {
    float pm[kBatch], pl[kBatch];
    float4 a[kBatch], b[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u;
      pm[u] = -INFINITY;
      pl[u] = 0.f;
      a[u] = b[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < pieces) {
        // Piece 0 lies in this CTA's second slot, piece i > 0 in CTA + i's first.
        const int64_t sl = 2 * (static_cast<int64_t>(blockIdx.x) + i) + (i == 0 ? 1 : 0);
        pm[u] = __ldcg(p.ml + sl * 512 + row);
        pl[u] = __ldcg(p.ml + sl * 512 + 256 + row);
        a[u] = __ldcg(p.part + (sl * (D / 4) + 2 * d8) * 256 + row);
        b[u] = __ldcg(p.part + (sl * (D / 4) + 2 * d8 + 1) * 256 + row);
      }
    }
    float mx = m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) mx = fmaxf(mx, pm[u]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float f = exp2_approx(m - ref);
    m = mx;
    den *= f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= f;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      f = exp2_approx(pm[u] - ref);
      den = fmaf(pl[u], f, den);
      const float v[8] = {a[u].x, a[u].y, a[u].z, a[u].w, b[u].x, b[u].y, b[u].z, b[u].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(v[e], f, acc[e]);
    }
  }
  const float inv = den == 0.f ? 0.f : __frcp_rn(den);
  uint4 w;
  uint32_t* ww = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
  for (int e = 0; e < 4; ++e) ww[e] = Elem<E>::pack(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  *reinterpret_cast<uint4*>(static_cast<E*>(p.out) +
                            (static_cast<int64_t>(tok0 + tok) * p.hq + kvh * p.g + r % p.g) * D + 8 * d8) = w;
}

template <typename E, int D>
cudaError_t launch(const Params& p, const CUtensorMap& qmap, const CUtensorMap& kmap,
                   const CUtensorMap& vmap, int num_sms, cudaStream_t stream) {
  static int configured[64] = {0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(prompt_kernel<E, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Layout<D>::kSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = 1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.splits && p.n_pieces < num_sms ? p.n_pieces : num_sms);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Layout<D>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, prompt_kernel<E, D>, p, qmap, kmap, vmap);
  if (e != cudaSuccess || p.splits) return e;
  cfg.gridDim = dim3(num_sms, 8);
  cfg.blockDim = dim3(32 * (D / 8));
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, prompt_join_kernel<E, D>, p);
}

size_t slot_bytes(int D) { return 256 * static_cast<size_t>(D) * 4 + 512 * 4; }
int pairs_of(int n, int tq) { return (n + 2 * tq - 1) / (2 * tq); }

}  // namespace

int prompt_box_rows(int page_size) { return page_size < kBlock ? page_size : kBlock; }
int prompt_tokens_per_tile(int hq, int n_kv_heads) { return 128 / (hq / n_kv_heads); }

size_t prompt_workspace(int D, int num_sms) {
  return static_cast<size_t>(num_sms) * (2 * slot_bytes(D) + sizeof(Desc));
}

// Pieces of a prefix: of 1 .. 64 a KV head and pair, those that keep the
// busiest SM's blocks fewest; half a block counted for each, for the joining.
int prefix_splits(int n_seqs, int hq, int n_kv_heads, int prefix_len, int num_sms) {
  const long long items = static_cast<long long>(pairs_of(n_seqs, prompt_tokens_per_tile(hq, n_kv_heads))) * n_kv_heads;
  const int blocks = (prefix_len + kBlock - 1) / kBlock;
  int best = 1;
  long long cost = -1;
  for (int s = 1; s <= 64 && s <= blocks; ++s) {
    const long long c = 2 * ((items * s + num_sms - 1) / num_sms * ((blocks + s - 1) / s)) + s;
    if (cost < 0 || c < cost) {
      cost = c;
      best = s;
    }
  }
  return best;
}

size_t prefix_workspace(int n_seqs, int hq, int n_kv_heads, int D, int prefix_len, int num_sms) {
  const size_t pieces = static_cast<size_t>(pairs_of(n_seqs, prompt_tokens_per_tile(hq, n_kv_heads))) * n_kv_heads *
                        prefix_splits(n_seqs, hq, n_kv_heads, prefix_len, num_sms);
  return pieces * slot_bytes(D);
}

PrefixPieces prefix_pieces(const PromptArgs& a, const PagedPool& pool, int num_sms) {
  PrefixPieces f;
  f.S = prefix_splits(a.T, a.hq, pool.n_kv_heads, a.prefix_len, num_sms);
  f.tq = prompt_tokens_per_tile(a.hq, pool.n_kv_heads);
  const size_t pieces = static_cast<size_t>(pairs_of(a.T, f.tq)) * pool.n_kv_heads * f.S;
  f.o = static_cast<const float*>(a.workspace);
  f.ml = f.o + pieces * 256 * pool.D;
  return f;
}

cudaError_t launch_prompt(const PagedPool& pool, const CUtensorMap& qmap, const CUtensorMap& kmap,
                          const CUtensorMap& vmap, const PromptArgs& a, int num_sms,
                          cudaStream_t stream) {
  Params p;
  p.v = pool.v;
  p.page_stride = pool.page_stride;
  p.head_stride = pool.head_stride;
  p.row_stride = pool.row_stride;
  p.table = a.table;
  p.q_starts = a.q_starts;
  p.lens = a.kv_lens;
  p.out = a.out;
  p.table_stride = a.table_stride;
  p.n_pages = pool.n_pages;
  p.B = a.B;
  p.T = a.T;
  p.hq = a.hq;
  p.hkv = pool.n_kv_heads;
  p.g = a.hq / pool.n_kv_heads;
  p.tq = prompt_tokens_per_tile(a.hq, pool.n_kv_heads);
  p.g_magic = p.g > 1 ? static_cast<uint32_t>(((uint64_t(1) << 32) + p.g - 1) / p.g) : 0;
  p.page_shift = 0;
  while ((1 << p.page_shift) < pool.page_size) ++p.page_shift;
  const int64_t limit = static_cast<int64_t>(a.table_width) * pool.page_size;
  p.len_limit = limit < (1 << 30) ? static_cast<int>(limit) : 1 << 30;
  p.box_rows = prompt_box_rows(pool.page_size);
  p.causal = a.causal;
  // (Each sequence for itself: starts that are out of order may count rows twice.)
  p.n_units32 = (static_cast<double>(a.T) / (2 * p.tq) + 1.0) * a.B * (static_cast<double>(p.len_limit) + kItemKeys) *
                    pool.n_kv_heads < 2147483648.0;
  p.scale_log2 = a.scale_log2;
  p.prefix_len = a.prefix_len;
  p.splits = p.n_pieces = 0;
  size_t slots = 2 * static_cast<size_t>(num_sms);
  if (a.prefix_len > 0) {
    p.causal = false;
    p.splits = prefix_splits(a.T, a.hq, pool.n_kv_heads, a.prefix_len, num_sms);
    slots = static_cast<size_t>(pairs_of(a.T, p.tq)) * pool.n_kv_heads * p.splits;
    p.n_pieces = static_cast<int>(slots);
  }
  p.part = static_cast<float4*>(a.workspace);
  p.ml = reinterpret_cast<float*>(p.part + slots * 64 * pool.D);
  p.desc = reinterpret_cast<Desc*>(p.ml + slots * 512);
  if (pool.bf16)
    return pool.D == 128 ? launch<__nv_bfloat16, 128>(p, qmap, kmap, vmap, num_sms, stream)
                         : launch<__nv_bfloat16, 64>(p, qmap, kmap, vmap, num_sms, stream);
  return pool.D == 128 ? launch<__half, 128>(p, qmap, kmap, vmap, num_sms, stream)
                       : launch<__half, 64>(p, qmap, kmap, vmap, num_sms, stream);
}

}  // namespace dqg

DQG_STATUS_READER(read_status_prompt)
