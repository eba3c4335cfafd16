"""Operators over a cache held in 8 bits, on the GPU, against plain 64-bit
restatements.

Stored blocks: the 16-bit values that the codes stand for are those that
``rope_paged_append`` writes for the same tokens (bit for bit). A scale is
max(fp32(max|x| / L), 2^-126) exactly. A code is fp32(L x / max|x|) rounded to
nearest, which is x / scale but for two fp32 roundings (the scale's and this), so
|code - x / scale| <= half a step + 2^-22 |x / scale|, a step being 1 (int8) or,
for e4m3, 2^-3 of the power of two at or below |x / scale|, 2^-9 at least.

Attention: outputs are rounded once to 16 bits (unit roundoff u = 2^-11 fp16,
2^-8 bf16) and each softmax weight once to 16 bits before the product with the
values, while the weights' sum is taken before: at most u * sum_j p_j |v_j| <= u
* max|v| per output. Exponentials and fp32 sums add below 2^-13 of that scale.
So |out - ref| <= u |ref| + (u + 2^-13) max|v|. Beside int8 codes the decode
step rounds queries to 2^-16 of their head's largest: a score changes by e <=
scale 2^-16 max|q| sum|k| (the sum over a key's values), a weight by a factor
within exp(2 e), an output by expm1(2 e) max|v| at most.
"""

from __future__ import annotations

import math

import pytest
import torch

from dequant_project_b200 import _native, paged_ops
from dequant_project_b200 import quantized_cache as qc

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float16, torch.bfloat16]
CODES = [torch.int8, torch.float8_e4m3fn]


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def make_cache(gen, lens, hkv, d, page, block, codes, dtype, device, extra=2, spread=0.5):
    """A cache whose complete blocks hold random codes and scales, with tables
    of scattered pages and open slots; whatever no position uses is NaN
    (scales, open rows, and e4m3 codes) or any code."""
    counts = [-(-n // page) for n in lens]
    n_pages, n_slots = sum(counts) + extra, len(lens) + 3
    order = torch.randperm(n_pages, generator=gen, device=device).int()
    table = torch.full((len(lens), max([1, *counts])), -1, dtype=torch.int32, device=device)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    slots = torch.randperm(n_slots, generator=gen, device=device)[:len(lens)].int()
    used = torch.zeros((n_pages, page), dtype=torch.bool, device=device)
    opened = torch.zeros((n_slots, block), dtype=torch.bool, device=device)
    for i, n in enumerate(lens):
        t = torch.arange(n - n % block, device=device)
        used[table[i].long()[t // page], t % page] = True
        opened[slots[i].long(), :n % block] = True
    parts = []
    for _ in range(2):
        raw = torch.randint(0, 256, (n_pages, hkv, page, d), generator=gen, device=device, dtype=torch.uint8)
        if codes == torch.float8_e4m3fn:
            raw[(raw & 0x7f) == 0x7f] -= 1  # no NaN among the codes in use
            raw.masked_fill_(~used[:, None, :, None], 0x7f)
        else:
            raw[raw == 0x80] = 0x81
        scale = torch.exp(spread * torch.randn((n_pages, hkv, page // block), generator=gen, device=device)) / 64
        if codes == torch.float8_e4m3fn:
            scale /= 4
        scale.masked_fill_(~used[:, ::block][:, None], float("nan"))
        opens = torch.randn((n_slots, hkv, block, d), generator=gen, device=device).to(dtype)
        opens.masked_fill_(~opened[:, None, :, None], float("nan"))
        parts.append((raw.view(codes), scale, opens))
    (k, ks, ko), (v, vs, vo) = parts
    return qc.QuantizedCache(k, v, ks, vs, ko, vo), table, slots


def rows64(cache, which, table_row, slot, n):
    """64-bit [n, kv heads, D]: the positions of one sequence."""
    codes, scale, opened = cache[which], cache[2 + which], cache[4 + which]
    page, block = cache.page_size, cache.block
    done = n - n % block
    t = torch.arange(done, device=codes.device)
    at = table_row.long()[t // page]
    x = codes.float()[at, :, t % page].double() * scale.double()[at, :, t % page // block][..., None]
    return torch.cat([x, opened[slot, :, :n - done].transpose(0, 1).double()])


def attend64(q, k, v, ends, scale):
    rows, hq, d = q.shape
    n, hkv, _ = k.shape
    if n == 0:
        return torch.zeros((rows, hq, d), dtype=torch.float64, device=q.device)
    s = torch.einsum("rkgd,tkd->rkgt", q.double().view(rows, hkv, hq // hkv, d), k) * scale
    hidden = torch.arange(n, device=q.device)[None] >= ends[:, None]
    s = s.masked_fill(hidden[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    return torch.einsum("rkgt,tkd->rkgd", p, v).reshape(rows, hq, d)


def check_attention(out, ref, v_max, dtype, e=0.0):
    u = U[dtype]
    err = (out.double() - ref).abs()
    lim = u * ref.abs() + (u + 2.0 ** -13 + math.expm1(2 * e)) * v_max + 1e-7
    assert bool((err <= lim).all()), f"max excess {float((err - lim).max()):.3e}, max error {float(err.max()):.3e}"


def clone(cache):
    return qc.QuantizedCache(*(t.clone() for t in cache))


def same_bits(a, b):
    return all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(a, b))


# ------------------------------------------------------------------- append
APPEND = [
    # new tokens, lengths with them, rows behind, hq, hkv, d, rotary dim, interleaved, norm, page, block
    ([1], [1], 0, 32, 32, 128, 128, False, False, 16, 16),
    ([1, 1, 1], [16, 33, 15], 0, 64, 8, 128, 128, False, True, 64, 16),
    ([40, 0, 3, 17], [40, 9, 18, 64], 5, 6, 2, 64, 64, True, False, 16, 16),
    ([100, 1], [131, 32], 0, 28, 4, 128, 32, False, True, 32, 32),
    ([9, 70], [9, 200], 2, 3, 1, 64, 24, False, True, 64, 64),     # partners cross lanes unevenly
    ([130], [190], 0, 4, 2, 128, 6, False, False, 256, 64),
    ([64, 63, 1], [128, 127, 64], 0, 8, 2, 128, 64, True, True, 64, 64),
    ([300, 7, 0], [300, 500, 0], 3, 33, 11, 64, 20, False, False, 16, 16),
    ([2] * 200, [17 + i % 40 for i in range(200)], 1, 4, 1, 64, 64, False, False, 32, 32),  # more than a block's threads
    ([31], [47], 0, 128, 1, 128, 128, False, False, 16, 16),
]


def append_case(gen, case, codes, dtype, device):
    new, lens, behind, hq, hkv, d, rot, inter, norm, page, block = case
    old = [n - q for q, n in zip(new, lens)]
    counts = [-(-n // page) for n in lens]
    n_pages = sum(counts) + 2
    order = torch.randperm(n_pages, generator=gen, device=device).int()
    table = torch.full((len(lens), max([1, *counts])), -1, dtype=torch.int32, device=device)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    cache = make_cache(gen, [0] * len(lens), hkv, d, page, block, codes, dtype, device, extra=n_pages)[0]
    for x in cache[4:]:  # open rows of earlier calls
        x.copy_(torch.randn(x.shape, generator=gen, device=device).to(dtype))
    slots = torch.randperm(cache.k_open.shape[0], generator=gen, device=device)[:len(lens)].int()
    t = sum(new) + behind
    positions = torch.randint(0, 4096, (t,), generator=gen, device=device)
    cos, sin = paged_ops.rope_scaled_tables(d, 10000.0, 4096, device, rotary_dim=rot)
    wide = torch.randn((t, (hq + 2 * hkv) * d + 8), generator=gen, device=device).to(dtype)
    qkv = wide[:, :-8]  # rows further apart than they are long
    qn = kn = None
    if norm:
        qn, kn = (1 + 0.1 * torch.randn((2, d), generator=gen, device=device)).to(dtype)
    starts = ints([0] + torch.tensor(new).cumsum(0).tolist(), device)
    return dict(qkv=qkv, cos=cos, sin=sin, positions=positions, cache=cache, block_table=table, open_slots=slots,
                q_starts=starts, kv_lens=ints(lens, device), n_q_heads=hq, interleaved=inter, q_norm=qn, k_norm=kn,
                eps=1e-5), old


def rows16(args):
    """Rotated queries, keys and values in 16 bits, by the 16-bit cache's append."""
    cache, t = args["cache"], args["qkv"].shape[0]
    hkv, d = cache.k.shape[1], cache.k.shape[3]
    pages = -(-max(t, 1) // 16)
    k, v = (torch.zeros((pages, hkv, 16, d), dtype=args["qkv"].dtype, device=args["qkv"].device) for _ in range(2))
    q = paged_ops.rope_paged_append(args["qkv"], args["cos"], args["sin"], args["positions"],
                                    torch.arange(t, device=k.device), k, v, args["n_q_heads"],
                                    interleaved=args["interleaved"], q_norm=args["q_norm"], k_norm=args["k_norm"],
                                    eps=args["eps"])
    return q, *(x.transpose(1, 2).reshape(-1, hkv, d)[:t] for x in (k, v))


def check_codes(codes, scale, x):
    """codes [hkv, block, D] and scale [hkv] against 16-bit values x."""
    most = qc.MOST[codes.dtype]
    # (Division in 64 bits and one rounding: torch divides fp32 CUDA tensors by a number with its reciprocal.)
    want = (x.double().abs().amax((1, 2)) / most).float().clamp(min=qc.LEAST_SCALE)
    assert torch.equal(scale, want)
    y = x.double() / scale.double()[:, None, None]
    step = torch.ones_like(y)
    if codes.dtype == torch.float8_e4m3fn:
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    err = (codes.float().double() - y).abs()
    assert bool((err <= step / 2 + 2.0 ** -22 * y.abs()).all()), float(err.max())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("case", APPEND, ids=lambda v: str(v)[:60])
def test_append(cuda_device, case, codes, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(sum(case[0]) + case[3])
    args, old = append_case(gen, case, codes, dtype, cuda_device)
    before = clone(args["cache"])
    q = qc.rope_quantized_append(**args)
    assert _native.device_status(cuda_device.index, reset=True) == 0
    rq, *rkv = rows16(args)
    assert torch.equal(q, rq)
    cache, table, slots = args["cache"], args["block_table"].long(), args["open_slots"].tolist()
    page, block = cache.page_size, cache.block
    wrote = torch.zeros(cache.k_scale.shape[0], cache.k_scale.shape[2], dtype=torch.bool, device=cuda_device)
    opened = torch.zeros(cache.k_open.shape[0], block, dtype=torch.bool, device=cuda_device)
    for b, (start, n, row) in enumerate(zip(old, case[1], args["q_starts"].tolist())):
        if n == start:
            continue
        for base in range(start - start % block, n, block):
            for which in (0, 1):
                lo, hi = max(base, start), min(base + block, n)
                new = rkv[which][row + lo - start:row + hi - start].transpose(0, 1)
                if hi == base + block:
                    x = torch.cat([before[4 + which][slots[b], :, :lo - base], new], 1)
                    at, part = table[b, base // page], base % page // block
                    check_codes(cache[which][at, :, base % page:base % page + block], cache[2 + which][at, :, part], x)
                    wrote[at, part] = True
                else:
                    assert torch.equal(cache[4 + which][slots[b], :, lo - base:hi - base], new)
                    opened[slots[b], lo - base:hi - base] = True
    for which in (0, 1):  # and nothing else
        now, then = (c[which].view(torch.uint8).unflatten(2, (-1, block)).transpose(1, 2) for c in (cache, before))
        assert torch.equal(now[~wrote], then[~wrote])
        now, then = (c[2 + which].view(torch.int32).transpose(1, 2) for c in (cache, before))
        assert torch.equal(now[~wrote], then[~wrote])
        now, then = (c[4 + which].view(torch.int16).transpose(1, 2) for c in (cache, before))
        assert torch.equal(now[~opened], then[~opened])


@pytest.mark.parametrize("block,page", [(16, 16), (32, 64), (64, 64)])
def test_a_cache_does_not_depend_on_how_a_prompt_was_cut(cuda_device, block, page):
    gen = torch.Generator(device=cuda_device).manual_seed(block)
    n, hq, hkv, d = 210, 4, 2, 128
    qkv = torch.randn((n, (hq + 2 * hkv) * d), generator=gen, device=cuda_device).half()
    cos, sin = paged_ops.rope_scaled_tables(d, 1e4, 256, cuda_device)
    table = torch.randperm(-(-n // page), generator=gen, device=cuda_device).int()[None]
    results = []
    for cuts in ([n], [1] * n, [5, 11, 16, 32, 1, 63, 64, 18], [200, 10]):
        cache = qc.QuantizedCache.empty(-(-n // page), hkv, page, d, 3, block=block, device=cuda_device)
        at = 0
        for c in cuts:
            rows = slice(at, at + c)
            at += c
            qc.rope_quantized_append(qkv[rows], cos, sin, torch.arange(n, device=cuda_device)[rows], cache, table,
                                     ints([1], cuda_device), ints([0, c], cuda_device), ints([at], cuda_device), hq)
        assert at == n
        # Rows of the open block behind the sequence's end hold what they held.
        for x in cache[4:]:
            x[1, :, n % block:] = 0
        results.append(cache)
    for other in results[1:]:
        assert same_bits(results[0], other)


def test_blocks_of_zeros_small_numbers_and_none_that_are_numbers(cuda_device):
    """Scales stay finite and positive; a value that is not finite makes its
    block (of its head, of keys or values) read as NaN and no other."""
    d, hq, hkv = 64, 2, 2
    cos, sin = paged_ops.rope_scaled_tables(d, 1e4, 64, cuda_device)
    qkv = torch.ones((64, (hq + 2 * hkv) * d), dtype=torch.bfloat16, device=cuda_device)
    k0, v0 = hq * d, (hq + hkv) * d
    qkv[:16, k0:k0 + d] = 0
    qkv[:16, v0:v0 + d] = 2.0 ** -133  # the smallest bf16 number
    qkv[20, v0 + 3] = float("inf")
    qkv[33, k0 + d + 5] = float("nan")
    for codes in CODES:
        cache = qc.QuantizedCache.empty(4, hkv, 16, d, 1, codes=codes, dtype=torch.bfloat16, device=cuda_device)
        args = (torch.zeros(64, dtype=torch.int64, device=cuda_device), cache, ints([[3, 1, 0, 2]], cuda_device),
                ints([0], cuda_device), ints([0, 64], cuda_device), ints([64], cuda_device))
        qc.rope_quantized_append(qkv, cos, sin, *args, hq)
        ks, vs = cache.k_scale[:, :, 0], cache.v_scale[:, :, 0]
        assert ks[3, 0] == 2.0 ** -126 and bool((cache.k[3, 0].float() == 0).all())
        assert vs[3, 0] == 2.0 ** -126 and bool((cache.v[3, 0].float() == 2.0 ** -7).all()) == (codes != torch.int8)
        bad_k, bad_v = (torch.zeros((4, hkv), dtype=torch.bool, device=cuda_device) for _ in range(2))
        bad_v[1, 0] = bad_k[0, 1] = True
        assert torch.equal(ks.isnan(), bad_k) and torch.equal(vs.isnan(), bad_v)
        assert bool((cache.v[1, 0].float() == 0).all())
        q = torch.ones((1, hq, d), dtype=torch.bfloat16, device=cuda_device)
        out = qc.quantized_attention(q, cache, *args[2:4], args[5])
        assert out.isnan().all()  # both heads see a block that is not a number
        out = qc.quantized_attention(q, cache, *args[2:4], ints([16], cuda_device))
        assert out.isfinite().all()
        k, v, _ = qc.expanded_pages(cache, *args[2:4], args[5], 4)
        assert torch.equal(k.isnan().all(-1).all(-1), bad_k[[3, 1, 0, 2]])
        assert torch.equal(v.isnan().any(-1).any(-1), bad_v[[3, 1, 0, 2]])


def test_append_leaves_out_what_is_out_of_range(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    cos, sin = paged_ops.rope_scaled_tables(64, 1e4, 8, cuda_device)
    cache = qc.QuantizedCache.empty(2, 2, 16, 64, 2, device=cuda_device)
    qkv = torch.randn((20, 8 * 64), generator=gen, device=cuda_device).half()
    positions = torch.zeros(20, dtype=torch.int64, device=cuda_device)
    good = dict(table=[[0, 1]], slots=[1], starts=[0, 20], lens=[20])
    for bad in (dict(table=[[0, 2]], lens=[32]), dict(table=[[-1, 2]]), dict(slots=[2]), dict(slots=[-1]),
                dict(starts=[0, 21]), dict(starts=[5, 3]), dict(starts=[-1, 3]), dict(lens=[19]), dict(lens=[33]),
                dict(lens=[-4])):
        c = {**good, **bad}
        before = clone(cache)
        q = qc.rope_quantized_append(qkv, cos, sin, positions, cache, ints(c["table"], cuda_device),
                                     ints(c["slots"], cuda_device), ints(c["starts"], cuda_device),
                                     ints(c["lens"], cuda_device), 4)
        assert torch.isfinite(q.float()).all()
        assert _native.device_status(cuda_device.index, reset=True) == 2, bad
        if "table" not in bad:
            assert same_bits(cache, before), bad
    positions[7], positions[9] = 8, -1
    qc.rope_quantized_append(qkv, cos, sin, positions, cache, ints([[0, 1]], cuda_device), ints([1], cuda_device),
                             ints([0, 20], cuda_device), ints([20], cuda_device), 4)
    assert _native.device_status(cuda_device.index, reset=True) == 2
    # The 200th of many sequences is looked at too.
    lens = [1] * 199 + [-1]
    qc.rope_quantized_append(qkv[:1], cos, sin, positions[:1], cache, ints([[0]] * 200, cuda_device),
                             ints([0] * 200, cuda_device), ints([0] + [1] * 200, cuda_device),
                             ints([1] + [0] * 198 + [1], cuda_device), 4)
    assert _native.device_status(cuda_device.index, reset=True) == 0
    qc.rope_quantized_append(qkv[:2], cos, sin, positions[:2], cache, ints([[0]] * 200, cuda_device),
                             ints([0] * 200, cuda_device), ints([0] + [1] * 199 + [2], cuda_device),
                             ints(lens, cuda_device), 4)
    assert _native.device_status(cuda_device.index, reset=True) == 2


# ------------------------------------------------------------------- expand
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("lens,hkv,d,page,block", [
    ([1], 1, 64, 16, 16), ([0, 5, 16, 0, 33, 200], 2, 128, 32, 16), ([64, 63, 65, 127], 3, 64, 64, 64),
    ([300, 1], 8, 128, 256, 32), ([17] * 300, 1, 64, 16, 16)], ids=lambda v: str(v)[:30])
def test_expand(cuda_device, lens, hkv, d, page, block, codes, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(sum(lens))
    cache, table, slots = make_cache(gen, lens, hkv, d, page, block, codes, dtype, cuda_device)
    counts = [-(-n // page) for n in lens]
    k, v, out = qc.expanded_pages(cache, table, slots, ints(lens, cuda_device), sum(counts))
    assert _native.device_status(cuda_device.index, reset=True) == 0
    assert out.shape == table.shape
    at = 0
    for b, (n, c) in enumerate(zip(lens, counts)):
        assert out[b, :c].tolist() == list(range(at, at + c))
        for which, pages in ((0, k), (1, v)):
            want = torch.zeros((c * page, hkv, d), dtype=torch.float64, device=cuda_device)
            want[:n] = rows64(cache, which, table[b], slots[b].long(), n)
            got = pages[at:at + c].transpose(1, 2).reshape(-1, hkv, d).double()
            # code * scale is rounded to fp32, and that to 16 bits: by u of itself, or, where fp16 has no
            # smaller steps than 2^-24 (below 2^-14; some products are 2^-17), by half of such a step.
            least = 2.0 ** -25 if dtype == torch.float16 else 0.0
            assert bool(((got - want).abs() <= (U[dtype] + 2.0 ** -23) * want.abs() + least).all())
        at += c
    # Without room for the last two pages: those are left out and reported.
    if sum(counts) > 2:
        _, _, out = qc.expanded_pages(cache, table, slots, ints(lens, cuda_device), sum(counts) - 2)
        assert _native.device_status(cuda_device.index, reset=True) == 2
        listed = torch.cat([out[b, :c] for b, c in enumerate(counts)])
        assert listed.tolist() == list(range(sum(counts) - 2)) + [-1, -1]


# ------------------------------------------------------------------- decode
DECODE = [
    # lengths, hq, hkv, d, page, block
    ([2049], 32, 32, 128, 16, 16),
    ([1], 32, 32, 128, 16, 16),
    ([0, 1, 63, 64, 65, 0, 127, 129], 64, 8, 128, 64, 16),
    ([300, 17, 0, 5000, 1, 64, 15, 16], 8, 1, 128, 64, 64),
    ([33, 1000, 257, 256, 255], 28, 4, 128, 128, 32),
    ([700, 2, 511], 16, 16, 64, 256, 16),
    ([129, 31, 90], 6, 2, 64, 32, 32),
    ([100, 2000], 40, 1, 64, 16, 16),      # three row blocks of query heads
    ([100, 1999], 24, 2, 128, 64, 64),     # twelve query heads a KV head
    ([75, 0], 128, 1, 128, 16, 16),
    ([0, 0, 0], 4, 2, 128, 16, 16),
    ([40] * 300, 2, 1, 64, 16, 16),        # more sequences than CTAs
    ([40] * 128, 64, 8, 128, 64, 32),      # many items of one tile
    ([64, 17] * 64, 128, 8, 128, 16, 16),
    ([63, 191, 1] * 60, 24, 4, 64, 64, 64),
]


def reference(q, cache, table, slots, lens, scale):
    return torch.cat([attend64(q[b:b + 1], *(rows64(cache, w, table[b], slots[b].long(), n) for w in (0, 1)),
                               torch.tensor([n], device=q.device), scale) for b, n in enumerate(lens)])


def largest_value(cache, table, slots, lens):
    return max([float(rows64(cache, 1, table[b], slots[b].long(), n).abs().max()) for b, n in enumerate(lens) if n],
               default=0.0)


def query_rounding(q, cache, table, slots, lens):
    """The bound e of how far rounded queries move a score."""
    if cache.k.dtype != torch.int8:
        return 0.0
    k = max([float(rows64(cache, 0, table[b], slots[b].long(), n).abs().sum(-1).max()) for b, n in enumerate(lens) if n],
            default=0.0)
    return 2.0 ** -16 * float(q.float().abs().max()) * k / math.sqrt(q.shape[2])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("lens,hq,hkv,d,page,block", DECODE, ids=lambda v: str(v)[:40])
def test_decode(cuda_device, lens, hq, hkv, d, page, block, codes, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(len(lens) + hq)
    cache, table, slots = make_cache(gen, lens, hkv, d, page, block, codes, dtype, cuda_device)
    q = torch.randn((len(lens), hq, d), generator=gen, device=cuda_device).to(dtype)
    kv_lens = ints(lens, cuda_device)
    out = qc.quantized_attention(q, cache, table, slots, kv_lens)
    assert _native.device_status(cuda_device.index, reset=True) == 0
    ref = reference(q, cache, table, slots, lens, 1 / math.sqrt(d))
    check_attention(out, ref, largest_value(cache, table, slots, lens), dtype, query_rounding(q, cache, table, slots, lens))
    ws = qc.quantized_attention_workspace(len(lens), hq, hkv, d, cuda_device).fill_(255)
    for _ in range(3):
        assert torch.equal(qc.quantized_attention(q, cache, table, slots, kv_lens, workspace=ws), out)


# ------------------------------------------------------------------- prompt
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("ql,kl,hq,hkv,d,page,block,codes", [
    ([1], [1], 4, 4, 128, 16, 16, torch.int8),
    ([300], [300], 16, 2, 128, 64, 32, torch.int8),
    ([40], [700], 8, 1, 128, 32, 16, torch.float8_e4m3fn),
    ([0, 5, 1, 0, 130, 64], [0, 5, 1, 9, 130, 64], 8, 2, 64, 64, 64, torch.float8_e4m3fn),
    ([7, 200], [3, 150], 4, 2, 128, 16, 16, torch.int8),      # more queries than keys: rows that see none
    ([33, 260], [33, 1000], 28, 4, 128, 256, 64, torch.int8),
], ids=lambda v: str(v)[:30])
def test_prompt(cuda_device, ql, kl, hq, hkv, d, page, block, codes, causal, dtype):
    """As the decode step, with exact queries, but values rounded to 16 bits:
    by u of themselves (or half of fp16's smallest step), below u max|v| in the
    output."""
    gen = torch.Generator(device=cuda_device).manual_seed(sum(ql) + hq)
    cache, table, slots = make_cache(gen, kl, hkv, d, page, block, codes, dtype, cuda_device)
    starts = ints([0] + torch.tensor(ql).cumsum(0).tolist(), cuda_device)
    q = torch.randn((sum(ql), hq, d), generator=gen, device=cuda_device).to(dtype)
    n_pages = sum(-(-n // page) for n in kl)
    out = qc.quantized_prompt_attention(q, cache, table, slots, starts, ints(kl, cuda_device), n_pages, causal=causal)
    assert _native.device_status(cuda_device.index, reset=True) == 0
    ws = qc.quantized_prompt_workspace(cache, len(kl), table.shape[1], n_pages).fill_(255)
    for _ in range(3):
        assert torch.equal(qc.quantized_prompt_attention(q, cache, table, slots, starts, ints(kl, cuda_device), n_pages,
                                                         causal=causal, workspace=ws), out)
    u = U[dtype]
    for b, (n_q, n) in enumerate(zip(ql, kl)):
        if n_q == 0:
            continue
        lo = int(starts[b])
        k, v = (rows64(cache, w, table[b], slots[b].long(), n) for w in (0, 1))
        ends = (n - n_q + torch.arange(n_q, device=cuda_device) + 1 if causal
                else torch.full((n_q,), n, device=cuda_device))
        ref = attend64(q[lo:lo + n_q], k, v, ends, 1 / math.sqrt(d))
        v_max = float(v.abs().max()) if n else 0.0
        lim = u * ref.abs() + (2 * u + 2.0 ** -13) * v_max + 2e-7
        assert bool(((out[lo:lo + n_q].double() - ref).abs() <= lim).all())


def test_operators_over_expanded_pages(cuda_device):
    """The 16-bit operators over expanded pages: keys rounded to 16 bits move a
    score by e <= u |q||k| / sqrt(d), and an output by expm1(2 e) max|v| at
    most; queries of the decode step as above."""
    gen = torch.Generator(device=cuda_device).manual_seed(12)
    kl = [300, 77]
    cache, table, slots = make_cache(gen, kl, 2, 128, 32, 16, torch.int8, torch.float16, cuda_device)
    starts, lens = ints([0, 200, 250], cuda_device), ints(kl, cuda_device)
    q = torch.randn((250, 8, 128), generator=gen, device=cuda_device).half()
    k, v, t = qc.expanded_pages(cache, table, slots, lens, 13)
    u, v_max = 2.0 ** -11, largest_value(cache, table, slots, kl)
    e = u * float(q.float().norm(dim=-1).max()) * float(k.float().norm(dim=-1).max()) / math.sqrt(128)
    want = paged_ops.prompt_attention(q, k, v, t, starts, lens)
    out = qc.quantized_prompt_attention(q, cache, table, slots, starts, lens, 13)
    assert float((out.float() - want.float()).abs().max()) <= (6 * u + 2.0 ** -12 + math.expm1(2 * e)) * v_max
    one = q[:2].contiguous()
    e += query_rounding(one, cache, table, slots, kl)
    a, b = qc.quantized_attention(one, cache, table, slots, lens), paged_ops.paged_attention(one, k, v, t, lens)
    assert float((a.float() - b.float()).abs().max()) <= (6 * u + 2.0 ** -12 + math.expm1(2 * e)) * v_max


def test_prompts_without_room_or_positions(cuda_device):
    """Pages that there is no room for are reported, and the other sequences are
    as they were; sequences without positions give zeros."""
    gen = torch.Generator(device=cuda_device).manual_seed(13)
    kl = [40, 3000, 0]
    cache, table, slots = make_cache(gen, kl, 2, 64, 16, 16, torch.int8, torch.float16, cuda_device)
    starts, lens = ints([0, 30, 60, 64], cuda_device), ints(kl, cuda_device)
    q = torch.randn((64, 4, 64), generator=gen, device=cuda_device).half()
    full = qc.quantized_prompt_attention(q, cache, table, slots, starts, lens, 191)
    assert _native.device_status(cuda_device.index, reset=True) == 0
    assert bool((full[60:] == 0).all())
    for n_pages in (3, 20):
        ws = qc.quantized_prompt_workspace(cache, 3, table.shape[1], n_pages).fill_(255)
        out = qc.quantized_prompt_attention(q, cache, table, slots, starts, lens, n_pages, workspace=ws)
        assert _native.device_status(cuda_device.index, reset=True) == 2
        assert torch.equal(out[:30], full[:30]) and bool((out[60:] == 0).all())
    none = qc.quantized_prompt_attention(q, cache, table, slots, starts, ints([0, 0, 0], cuda_device), 0)
    assert bool((none == 0).all())
    assert _native.device_status(cuda_device.index, reset=True) == 0
