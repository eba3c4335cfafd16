"""Paged-cache operators on the GPU against plain 64-bit restatements.

Tolerances follow from the kernels' arithmetic. Outputs are rounded once to
16 bits (unit roundoff u = 2^-11 fp16, 2^-8 bf16). Attention also rounds each
softmax weight to 16 bits before the product with the values, while the weights'
sum is taken before rounding: that is at most u * sum_j p_j |v_j| <= u * max|v|
per output. Exponentials and fp32 sums add below 2^-13 of that scale. So
|out - ref| <= u |ref| + (u + 2^-13) max|v|.
"""

from __future__ import annotations

import math

import pytest
import torch

from dequant_project_b200 import _native, paged_ops

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float16, torch.bfloat16]


def make_cache(gen, lens, hkv, d, page, dtype, device, width=None, extra=2, fill=None):
    """Pools and table of scattered pages; whatever no position uses is
    ``fill`` (random numbers by default)."""
    counts = [-(-n // page) for n in lens]
    n_pages = sum(counts) + extra
    order = torch.randperm(n_pages, generator=gen, device=device).int()
    table = torch.full((len(lens), max([1, *counts]) if width is None else width), -1, dtype=torch.int32,
                       device=device)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    k = torch.randn((n_pages, hkv, page, d), generator=gen, device=device).to(dtype)
    v = torch.randn((n_pages, hkv, page, d), generator=gen, device=device).to(dtype)
    if fill is not None:
        used = torch.zeros((n_pages, page), dtype=torch.bool, device=device)
        for i, n in enumerate(lens):
            t = torch.arange(n, device=device)
            used[table[i].long()[t // page], t % page] = True
        mask = ~used[:, None, :, None]
        k.masked_fill_(mask, fill)
        v.masked_fill_(mask, fill)
    return k, v, table


def rows64(pages, table_row, n):
    page = pages.shape[2]
    t = torch.arange(n, device=pages.device)
    return pages[table_row.long()[t // page], :, t % page].double()  # [n, hkv, d]


def attend64(q, k, v, ends, scale):
    """q [rows, hq, d] over k, v [n, hkv, d] in 64 bits, row by row's end."""
    rows, hq, d = q.shape
    n, hkv, _ = k.shape
    g = hq // hkv
    out = torch.zeros((rows, hq, d), dtype=torch.float64, device=q.device)
    if n == 0:
        return out
    s = torch.einsum("rkgd,tkd->rkgt", q.double().view(rows, hkv, g, d), k) * scale
    hidden = torch.arange(n, device=q.device)[None] >= ends[:, None]
    s = s.masked_fill(hidden[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    return torch.einsum("rkgt,tkd->rkgd", p, v).reshape(rows, hq, d)


def check_attention(out, ref, v_max, dtype):
    u = U[dtype]
    err = (out.double() - ref).abs()
    lim = u * ref.abs() + (u + 2.0 ** -13) * v_max + 1e-7
    assert bool((err <= lim).all()), f"max excess {float((err - lim).max()):.3e}, max error {float(err.max()):.3e}"


# ------------------------------------------------------------------- append
def append64(qkv, cos, sin, positions, hq, hkv, d, interleaved, qn, kn, eps):
    t = qkv.shape[0]
    x = qkv.double().view(t, hq + 2 * hkv, d)
    h = x[:, :hq + hkv].clone()
    if qn is not None:
        w = torch.cat([qn.double().expand(hq, d), kn.double().expand(hkv, d)])
        h = h / torch.sqrt((h ** 2).mean(-1, keepdim=True) + eps) * w
    n = cos.shape[1]
    i = torch.arange(n, device=qkv.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    o = h.clone()
    o[..., a] = h[..., a] * c - h[..., b] * s
    o[..., b] = h[..., b] * c + h[..., a] * s
    return o[:, :hq], o[:, hq:], x[:, hq + hkv:]


APPEND = [
    # tokens, hq, hkv, d, rotary dim, interleaved, norm, page, every n-th skipped
    (1, 32, 32, 128, 128, False, False, 16, 0),
    (5, 64, 8, 128, 128, False, True, 64, 0),
    (33, 6, 2, 64, 64, True, False, 16, 3),
    (17, 28, 4, 128, 32, False, True, 32, 4),
    (9, 3, 1, 64, 24, False, True, 16, 0),    # partners cross lanes unevenly
    (9, 3, 1, 128, 6, False, False, 256, 2),
    (7, 4, 4, 64, 2, True, True, 128, 0),
    (700, 32, 8, 128, 64, True, True, 16, 7),  # several heads a lane group
    (700, 33, 11, 64, 20, False, False, 16, 0),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append(cuda_device, case, dtype):
    t, hq, hkv, d, rot, inter, norm, page, skip = case
    gen = torch.Generator(device=cuda_device).manual_seed(t + hq)
    k, v, table = make_cache(gen, [t], hkv, d, page, dtype, cuda_device)
    k0, v0 = k.clone(), v.clone()
    at = torch.arange(t, device=cuda_device)
    slots = table[0].long()[at // page] * page + at % page
    if skip:
        slots[::skip] = -1
    positions = torch.randint(0, 4096, (t,), generator=gen, device=cuda_device)
    cos, sin = paged_ops.rope_scaled_tables(d, 10000.0, 4096, cuda_device, rotary_dim=rot)
    wide = torch.randn((t, (hq + 2 * hkv) * d + 8), generator=gen, device=cuda_device).to(dtype)
    qkv = wide[:, :-8]  # rows further apart than they are long
    qn = kn = None
    if norm:
        qn, kn = (1 + 0.1 * torch.randn((2, d), generator=gen, device=cuda_device)).to(dtype)
    q = paged_ops.rope_paged_append(qkv, cos, sin, positions, slots, k, v, hq, interleaved=inter, q_norm=qn,
                                    k_norm=kn, eps=1e-5)
    rq, rk, rv = append64(qkv, cos, sin, positions, hq, hkv, d, inter, qn, kn, 1e-5)
    # One rounding of a value formed in fp32 from at most six operations on
    # normed values of size up to |y|: u |ref| + 2^-20 max|y|.
    u = U[dtype]
    scale = max(float(rq.abs().max()), float(rk.abs().max()))
    for got, ref in ((q, rq),):
        assert bool(((got.double() - ref).abs() <= u * ref.abs() + 2.0 ** -20 * scale).all())
    kept = slots >= 0
    ek, ev = k0.double(), v0.double()
    sl = slots[kept]
    ek[sl // page, :, sl % page] = rk[kept]
    ev[sl // page, :, sl % page] = rv[kept]
    assert bool(((k.double() - ek).abs() <= u * ek.abs() + 2.0 ** -20 * scale).all())
    assert torch.equal(v.double(), ev)
    written = torch.zeros((k.shape[0], page), dtype=torch.bool, device=cuda_device)
    written[sl // page, sl % page] = True
    untouched = ~written[:, None, :, None].expand_as(k)
    assert torch.equal(k[untouched], k0[untouched])
    assert _native.device_status(cuda_device.index) == 0


def test_append_leaves_out_what_is_out_of_range(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    k, v, _ = make_cache(gen, [16], 2, 64, 16, torch.float16, cuda_device, extra=1)
    k0, v0 = k.clone(), v.clone()
    cos, sin = paged_ops.rope_scaled_tables(64, 1e4, 8, cuda_device)
    qkv = torch.randn((3, 8 * 64), generator=gen, device=cuda_device).half()
    slots = torch.tensor([32, 1 << 40, -5], device=cuda_device)  # the pool has 32 slots
    positions = torch.tensor([0, 9, -1], device=cuda_device)
    q = paged_ops.rope_paged_append(qkv, cos, sin, positions, slots, k, v, 4)
    assert torch.isfinite(q.float()).all()
    assert torch.equal(k, k0) and torch.equal(v, v0)
    assert _native.device_status(cuda_device.index, reset=True) == 2
    assert _native.device_status(cuda_device.index) == 0


def test_append_on_one_buffer_of_keys_and_values(cuda_device):
    """Pools that are views of one [pages, 2, heads, page, D] allocation."""
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    both = torch.randn((4, 2, 2, 16, 128), generator=gen, device=cuda_device).half()
    flat = both.clone()
    k, v = both[:, 0], both[:, 1]
    cos, sin = paged_ops.rope_scaled_tables(128, 1e4, 64, cuda_device)
    qkv = torch.randn((20, 8 * 128), generator=gen, device=cuda_device).half()
    pos = torch.arange(20, device=cuda_device)
    slots = pos + 16
    paged_ops.rope_paged_append(qkv, cos, sin, pos, slots, k, v, 4)
    kc, vc = flat[:, 0].contiguous(), flat[:, 1].contiguous()
    paged_ops.rope_paged_append(qkv, cos, sin, pos, slots, kc, vc, 4)
    assert torch.equal(k, kc) and torch.equal(v, vc)


# ------------------------------------------------------------------- decode
DECODE = [
    # lengths, hq, hkv, d, page
    ([2049], 32, 32, 128, 16),
    ([1], 32, 32, 128, 16),
    ([0, 1, 63, 64, 65, 0, 127, 129], 64, 8, 128, 16),
    ([300, 17, 0, 5000, 1, 64], 8, 1, 128, 64),
    ([33, 1000, 257, 256, 255], 28, 4, 128, 128),
    ([700, 2, 511], 16, 16, 64, 256),
    ([129, 31, 90], 6, 2, 64, 32),
    ([100, 2000], 40, 1, 64, 16),      # three row blocks of query heads
    ([75, 0], 128, 1, 128, 16),
    ([0, 0, 0], 4, 2, 128, 16),
    ([40] * 300, 2, 1, 64, 16),        # more sequences than CTAs
    ([40] * 128, 64, 8, 128, 64),      # many items of one tile: queries' places are soon reused
    ([64, 17] * 64, 128, 8, 128, 16),
    ([33] * 200, 24, 4, 64, 32),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lens,hq,hkv,d,page", DECODE, ids=lambda v: str(v)[:40])
def test_decode(cuda_device, lens, hq, hkv, d, page, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(len(lens) + hq)
    k, v, table = make_cache(gen, lens, hkv, d, page, dtype, cuda_device, fill=float("nan"))
    q = torch.randn((len(lens), hq, d), generator=gen, device=cuda_device).to(dtype)
    kv_lens = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    out = paged_ops.paged_attention(q, k, v, table, kv_lens)
    scale = 1 / math.sqrt(d)
    v_max = float(torch.nan_to_num(v.float()).abs().max())
    ref = torch.cat([attend64(q[i:i + 1], rows64(k, table[i], n), rows64(v, table[i], n),
                              kv_lens[i:i + 1], scale) for i, n in enumerate(lens)])
    check_attention(out, ref, v_max, dtype)
    ws = paged_ops.paged_attention_workspace(len(lens), hq, hkv, d, cuda_device).fill_(255)
    for _ in range(3):
        assert torch.equal(paged_ops.paged_attention(q, k, v, table, kv_lens, workspace=ws), out)
    assert _native.device_status(cuda_device.index) == 0


# ------------------------------------------------------------------- prompt
def prompt_case(gen, q_lens, kv_lens, hq, hkv, d, page, dtype, device, fill=float("nan")):
    k, v, table = make_cache(gen, kv_lens, hkv, d, page, dtype, device, fill=fill)
    starts = torch.tensor([0] + q_lens, device=device).cumsum(0).int()
    q = torch.randn((int(starts[-1]), hq, d), generator=gen, device=device).to(dtype)
    return q, k, v, table, starts, torch.tensor(kv_lens, dtype=torch.int32, device=device)


def prompt64(q, k, v, table, starts, kv_lens, causal, scale):
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for i in range(len(kv_lens)):
        lo, hi, n = int(starts[i]), int(starts[i + 1]), int(kv_lens[i])
        ends = (n - (hi - lo) + torch.arange(hi - lo, device=q.device) + 1 if causal
                else torch.full((hi - lo,), n, device=q.device))
        if hi > lo and n:
            out[lo:hi] = attend64(q[lo:hi], rows64(k, table[i], n), rows64(v, table[i], n), ends, scale)
    return out


PROMPT = [
    # query lengths, key lengths, hq, hkv, d, page
    ([1], [1], 4, 4, 128, 16),
    ([128], [128], 2, 2, 128, 128),
    ([257], [257], 3, 3, 128, 64),
    ([300], [300], 16, 2, 128, 16),
    ([40], [700], 8, 1, 128, 32),             # a chunk: few rows, many keys
    ([1], [5000], 64, 8, 128, 64),            # one row, cut over many CTAs
    ([0, 5, 1, 0, 130, 64], [0, 5, 1, 9, 130, 64], 8, 2, 64, 16),
    ([7, 200], [3, 150], 4, 2, 128, 16),      # more queries than keys: rows that see none
    ([3], [0], 4, 2, 128, 16),
    ([33, 260], [33, 1000], 28, 4, 128, 256),  # 7 heads a group: 126 of a tile's rows
    ([19], [90], 48, 1, 64, 32),              # 96 of 128 rows
    ([5], [300], 128, 1, 128, 128),
    ([9], [40], 100, 1, 128, 16),
    ([700, 1, 513], [700, 800, 600], 6, 3, 64, 128),
    ([1] * 200, list(range(1, 201)), 4, 2, 128, 16),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("ql,kl,hq,hkv,d,page", PROMPT, ids=lambda v: str(v)[:40])
def test_prompt(cuda_device, ql, kl, hq, hkv, d, page, causal, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(sum(ql) + hq)
    args = prompt_case(gen, ql, kl, hq, hkv, d, page, dtype, cuda_device)
    out = paged_ops.prompt_attention(*args, causal=causal)
    assert _native.device_status(cuda_device.index, reset=True) == 0
    ref = prompt64(*args, causal, 1 / math.sqrt(d))
    check_attention(out, ref, float(torch.nan_to_num(args[2].float()).abs().max()), dtype)
    ws = paged_ops.prompt_attention_workspace(d, cuda_device).fill_(255)
    for _ in range(3):
        assert torch.equal(paged_ops.prompt_attention(*args, causal=causal, workspace=ws), out)


# ------------------------------------------------------------ shared prefix
PREFIX = [
    # prefix, own lengths, hq, hkv, d, page
    (1, [0, 5, 70], 8, 2, 128, 16),
    (130, [0, 0], 4, 4, 128, 64),
    (2000, [1, 300, 0, 64, 65], 32, 32, 128, 16),
    (777, [30] * 50, 64, 8, 128, 32),
    (5000, [100, 3], 28, 4, 128, 128),
    (300, [9, 0, 200], 40, 1, 64, 16),
    (0, [9, 0, 200], 8, 2, 64, 256),
    (900, [1], 100, 1, 64, 16),
    (128, list(range(300)), 2, 2, 64, 16),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("prefix,lens,hq,hkv,d,page", PREFIX, ids=lambda v: str(v)[:40])
def test_shared_prefix(cuda_device, prefix, lens, hq, hkv, d, page, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(prefix + hq)
    k, v, table = make_cache(gen, lens + [prefix], hkv, d, page, dtype, cuda_device, fill=float("nan"))
    own, shared = table[:-1].contiguous(), table[-1].contiguous()
    q = torch.randn((len(lens), hq, d), generator=gen, device=cuda_device).to(dtype)
    kv_lens = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    out = paged_ops.shared_prefix_attention(q, k, v, shared, prefix, own, kv_lens)
    assert _native.device_status(cuda_device.index, reset=True) == 0
    ref = []
    for i, n in enumerate(lens):
        kk, vv = (torch.cat([rows64(p, shared, prefix), rows64(p, own[i], n)]) for p in (k, v))
        ref.append(attend64(q[i:i + 1], kk, vv, kv_lens[i:i + 1] + prefix, 1 / math.sqrt(d)))
    check_attention(out, torch.cat(ref), float(torch.nan_to_num(v.float()).abs().max()), dtype)
    for _ in range(3):
        assert torch.equal(paged_ops.shared_prefix_attention(q, k, v, shared, prefix, own, kv_lens), out)


# ------------------------------------------- values, layouts, streams, limits
def _growing(k, table, lens, page, per_block):
    """Keys whose size grows along each sequence, so that the running maximum
    moves in every block."""
    for i, n in enumerate(lens):
        t = torch.arange(n, device=k.device)
        f = (per_block ** (t // 64)).to(k.dtype)
        k[table[i].long()[t // page], :, t % page] *= f[:, None, None]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_maximum_that_keeps_growing(cuda_device, dtype):
    """Scores grow from block to block by more than the factor at which the
    accumulators are rescaled. Scores up to |s| = 2^6 carry an error of about
    2^-19 of fp32 sums, so the bound above holds as it is."""
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    lens, hq, hkv, d, page = [700, 130], 8, 2, 128, 16
    args = list(prompt_case(gen, [300, 130], lens, hq, hkv, d, page, dtype, cuda_device))
    _growing(args[1], args[3], lens, page, 1.2)
    q, k, v, table, starts, kv_lens = args
    v_max = float(torch.nan_to_num(v.float()).abs().max())
    out = paged_ops.prompt_attention(*args)
    check_attention(out, prompt64(*args, True, 1 / math.sqrt(d)), v_max, dtype)
    qd = q[:2].contiguous()
    ref = torch.cat([attend64(qd[i:i + 1], rows64(k, table[i], n), rows64(v, table[i], n), kv_lens[i:i + 1],
                              1 / math.sqrt(d)) for i, n in enumerate(lens)])
    check_attention(paged_ops.paged_attention(qd, k, v, table, kv_lens), ref, v_max, dtype)


def test_scale_is_taken(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(6)
    args = prompt_case(gen, [70], [200], 4, 2, 64, 16, torch.float16, cuda_device)
    q, k, v, table, starts, lens = args
    out = paged_ops.prompt_attention(*args, scale=0.4)
    check_attention(out, prompt64(*args, True, 0.4), 6.0, torch.float16)
    out = paged_ops.paged_attention(q[:1], k, v, table, lens, scale=0.4)
    ref = attend64(q[:1], rows64(k, table[0], 200), rows64(v, table[0], 200), lens, 0.4)
    check_attention(out, ref, 6.0, torch.float16)


def test_non_finite_keys_and_values(cuda_device):
    """A NaN or infinity that a row sees reaches it as in the formula; other
    sequences, and rows whose mask hides a NaN key, do not notice."""
    gen = torch.Generator(device=cuda_device).manual_seed(7)
    lens = [90, 90, 90, 150]
    args = prompt_case(gen, [90, 90, 90, 150], lens, 2, 2, 128, 16, torch.float16, cuda_device)
    q, k, v, table, starts, kv_lens = args
    clean = paged_ops.prompt_attention(*args)
    k2, v2 = k.clone(), v.clone()
    k2[table[0, 40 // 16], :, 40 % 16] = float("nan")   # seen by rows 40.. of sequence 0
    v2[table[1, 0], :, 0, 5] = float("inf")             # seen by every row of sequence 1
    out = paged_ops.prompt_attention(q, k2, v2, table, starts, kv_lens)
    assert torch.equal(out[:40], clean[:40])
    assert torch.isnan(out[40:90]).all()
    assert torch.isinf(out[90:180, :, 5]).all()
    keep = [i for i in range(128) if i != 5]
    assert torch.equal(out[90:180][..., keep], clean[90:180][..., keep])
    assert torch.equal(out[180:], clean[180:])
    qd = q[[0, 90, 180, 270]].contiguous()
    plain = paged_ops.paged_attention(qd, k, v, table, kv_lens)
    out = paged_ops.paged_attention(qd, k2, v2, table, kv_lens)
    assert torch.isnan(out[0]).all() and torch.isinf(out[1, :, 5]).all()
    assert torch.equal(out[2:], plain[2:])


@pytest.mark.parametrize("d", [64, 128])
def test_strided_inputs(cuda_device, d):
    """Queries as a view of a wider projection, keys and values as views of one
    buffer with rows further apart, a table that is part of a wider one."""
    gen = torch.Generator(device=cuda_device).manual_seed(8)
    hq, hkv, page, lens, ql = 8, 2, 16, [100, 37, 64], [30, 37, 1]
    k, v, table = make_cache(gen, lens, hkv, d, page, torch.float16, cuda_device, width=12)
    both = torch.randn((k.shape[0], page, 2 * hkv, d + 8), generator=gen, device=cuda_device).half()
    kv, vv = (both[:, :, i * hkv:(i + 1) * hkv, :d].permute(0, 2, 1, 3) for i in (0, 1))
    kv.copy_(k)
    vv.copy_(v)
    wide = torch.randn((sum(ql), hq * d + 64), generator=gen, device=cuda_device).half()
    q = wide[:, 64:].unflatten(1, (hq, d))
    starts = torch.tensor([0, 30, 67, 68], dtype=torch.int32, device=cuda_device)
    kv_lens = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    part = table[:, :7]
    want = paged_ops.prompt_attention(q.contiguous(), k, v, table, starts, kv_lens)
    assert torch.equal(paged_ops.prompt_attention(q, kv, vv, part, starts, kv_lens), want)
    want = paged_ops.paged_attention(q[:3].contiguous(), k, v, table, kv_lens)
    assert torch.equal(paged_ops.paged_attention(q[:3], kv, vv, part, kv_lens), want)
    pre = table[0, :3].contiguous()
    for n in (3, 60):  # streamed with the sequences; by the prompt kernel
        rows = q[:n] if n == 3 else q
        tab = part if n == 3 else part[:1].expand(68, 7).contiguous()
        ln = kv_lens if n == 3 else kv_lens[:1].expand(68).contiguous()
        want = paged_ops.shared_prefix_attention(rows.contiguous(), k, v, pre, 40, tab, ln)
        assert torch.equal(paged_ops.shared_prefix_attention(rows, kv, vv, pre, 40, tab, ln), want)


def test_offsets_past_32_bits(cuda_device):
    """Pages 2^28 elements apart: offsets past 2^31 elements and 2^32 bytes."""
    gen = torch.Generator(device=cuda_device).manual_seed(9)
    hkv, page, d, n = 2, 16, 128, 12
    k, v, table = make_cache(gen, [150], hkv, d, page, torch.float16, cuda_device)
    span = 1 << 28
    big = torch.empty(n * span, dtype=torch.float16, device=cuda_device)
    strides = (span, page * d, d, 1)
    kb = torch.as_strided(big, (n, hkv, page, d), strides)
    vb = torch.as_strided(big, (n, hkv, page, d), strides, 1 << 20)
    kb[:k.shape[0]].copy_(k)
    vb[:k.shape[0]].copy_(v)
    move = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=cuda_device)  # the far end holds page 0
    kb.copy_(kb.clone()[move.long()])
    vb.copy_(vb.clone()[move.long()])
    far = move[table.long().clamp(min=0)]
    lens = torch.tensor([150], dtype=torch.int32, device=cuda_device)
    starts = torch.tensor([0, 20], dtype=torch.int32, device=cuda_device)
    q = torch.randn((20, 4, d), generator=gen, device=cuda_device).half()
    assert torch.equal(paged_ops.prompt_attention(q, kb, vb, far, starts, lens),
                       paged_ops.prompt_attention(q, k, v, table, starts, lens))
    assert torch.equal(paged_ops.paged_attention(q[:1], kb, vb, far, lens),
                       paged_ops.paged_attention(q[:1], k, v, table, lens))
    cos, sin = paged_ops.rope_scaled_tables(d, 1e4, 64, cuda_device)
    qkv = torch.randn((16, 8 * d), generator=gen, device=cuda_device).half()
    pos = torch.arange(16, device=cuda_device)
    paged_ops.rope_paged_append(qkv, cos, sin, pos, pos + 16 * (n - 1), kb, vb, 4)
    paged_ops.rope_paged_append(qkv, cos, sin, pos, pos, k, v, 4)
    assert torch.equal(kb[n - 1], k[0]) and torch.equal(vb[n - 1], v[0])


def test_pages_may_lie_anywhere(cuda_device):
    """The same sequence through other pages, another page size and another
    place in the batch gives the same bits where the shares are cut alike."""
    gen = torch.Generator(device=cuda_device).manual_seed(10)
    k, v, table = make_cache(gen, [200, 200], 2, 128, 16, torch.bfloat16, cuda_device)
    t = torch.arange(200, device=cuda_device)
    for pool in (k, v):  # the second sequence holds what the first does
        pool[table[1].long()[t // 16], :, t % 16] = pool[table[0].long()[t // 16], :, t % 16]
    q = torch.randn((1, 8, 128), generator=gen, device=cuda_device).bfloat16()
    one = torch.tensor([200], dtype=torch.int32, device=cuda_device)
    a = paged_ops.paged_attention(q, k, v, table[:1], one)
    assert torch.equal(paged_ops.paged_attention(q, k, v, table[1:], one), a)


def test_captured_calls_serve_other_lengths(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(11)
    lens = [500, 300, 800]
    k, v, table = make_cache(gen, lens, 2, 128, 16, torch.float16, cuda_device)
    q = torch.randn((3, 8, 128), generator=gen, device=cuda_device).half()
    kv_lens = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    starts = torch.tensor([0, 1, 1, 3], dtype=torch.int32, device=cuda_device)
    pre = table[2, :4].contiguous()

    def calls():
        return (paged_ops.paged_attention(q, k, v, table, kv_lens),
                paged_ops.prompt_attention(q, k, v, table, starts, kv_lens),
                paged_ops.shared_prefix_attention(q, k, v, pre, 60, table, kv_lens))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = calls()
    for new in ([500, 300, 800], [1, 0, 799], [64, 65, 63]):
        kv_lens.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, calls()):
            assert torch.equal(a, b), new


def test_on_another_stream(cuda_device):
    """Work is queued on torch's current stream: behind what fills the inputs
    there, and not on the default stream."""
    gen = torch.Generator(device=cuda_device).manual_seed(12)
    k, v, table = make_cache(gen, [600], 2, 128, 16, torch.float16, cuda_device)
    q = torch.randn((1, 4, 128), generator=gen, device=cuda_device).half()
    lens = torch.tensor([600], dtype=torch.int32, device=cuda_device)
    want = paged_ops.paged_attention(q, k, v, table, lens)
    late = torch.zeros_like(q)
    big = torch.randn((4096, 4096), device=cuda_device)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(4):
            big = big @ big
            big = big / big.abs().max()
        late.copy_(q)
        out = paged_ops.paged_attention(late, k, v, table, lens)
    s.synchronize()
    assert torch.equal(out, want)


def test_indexes_out_of_range_are_left_out(cuda_device):
    """A page number no page has reads as zeros, a length past the table ends at
    it; both are reported, and nothing else is touched."""
    gen = torch.Generator(device=cuda_device).manual_seed(13)
    k, v, table = make_cache(gen, [64, 64], 2, 128, 16, torch.float16, cuda_device)
    q = torch.randn((2, 4, 128), generator=gen, device=cuda_device).half()
    lens = torch.tensor([64, 64], dtype=torch.int32, device=cuda_device)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda_device)
    calls = [lambda t, n: paged_ops.paged_attention(q, k, v, t, n),
             lambda t, n: paged_ops.prompt_attention(q, k, v, t, starts, n)]
    for call in calls:
        good = call(table, lens)
        for bad in (-7, 1 << 30, k.shape[0]):
            t = table.clone()
            t[0, 2] = bad
            out = call(t, lens)
            assert torch.equal(out[1], good[1]) and torch.isfinite(out).all()
            assert _native.device_status(cuda_device.index, reset=True) == 2
        for n in (65, 1 << 30, -3):
            out = call(table, torch.tensor([n, 64], dtype=torch.int32, device=cuda_device))
            assert torch.equal(out[1], good[1])
            assert torch.equal(out[0], good[0] if n > 0 else torch.zeros_like(out[0]))
            assert _native.device_status(cuda_device.index, reset=True) == 2
    # Starts out of order: those sequences have no rows.
    wrong = torch.tensor([0, 5, 2], dtype=torch.int32, device=cuda_device)
    paged_ops.prompt_attention(q, k, v, table, wrong, lens)
    torch.cuda.synchronize()
    assert _native.device_status(cuda_device.index, reset=True) in (0, 2)


def test_empty_calls(cuda_device):
    k = torch.zeros((2, 1, 16, 64), dtype=torch.float16, device=cuda_device)
    q = torch.zeros((0, 2, 64), dtype=torch.float16, device=cuda_device)
    none = torch.zeros((0, 1), dtype=torch.int32, device=cuda_device)
    lens = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    starts = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    assert paged_ops.paged_attention(q, k, k, none, lens).shape == (0, 2, 64)
    assert paged_ops.prompt_attention(q, k, k, none, starts, lens).shape == (0, 2, 64)
    pre = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    assert paged_ops.shared_prefix_attention(q, k, k, pre, 3, none, lens).shape == (0, 2, 64)


def test_binding_rejects_bad_tensors(cuda_device):
    def z(*shape, dtype=torch.float16, device=cuda_device):
        return torch.zeros(shape, dtype=dtype, device=device)

    k, q, t, n = z(2, 1, 16, 64), z(3, 2, 64), z(3, 2, dtype=torch.int32), z(3, dtype=torch.int32)
    cases = [
        ((q.float(), k, k, t, n), "q must be float16"),
        ((q.bfloat16(), k, k, t, n), "q must be float16"),
        ((q, k.float(), k.float(), t, n), "pages must be float16 or bfloat16"),
        ((q, k[0], k[0], t, n), "pages must be"),
        ((q, k, z(2, 1, 32, 64), t, n), "one shape, type and strides"),
        ((q, k, k.transpose(2, 3).contiguous().transpose(2, 3), t, n), "one shape, type and strides"),
        ((q, k, k.cpu(), t, n), "same device"),
        ((q, k, k, t.cpu(), n), "block_table must be"),
        ((q, k, k, t.long(), n), "block_table must be"),
        ((q, k, k, t[:2], n), "block_table must hold 3 rows"),
        ((q, k, k, t, n.long()), "kv_lens must be"),
        ((q, k, k, t, n[:1]), "kv_lens must hold 3 rows"),
        ((q[:, :, :32], k, k, t, n), "q must be"),
        ((q.transpose(1, 2).contiguous().transpose(1, 2), k, k, t, n), "head dimension contiguous"),
        ((z(3, 2, 96), z(2, 1, 16, 96), z(2, 1, 16, 96), t, n), "head_dim 64 and 128"),
        ((q, z(2, 1, 24, 64), z(2, 1, 24, 64), t, n), "page_size must be"),
        ((q, z(2, 3, 16, 64), z(2, 3, 16, 64), t, n), "query heads per KV head"),
    ]
    for args, msg in cases:
        with pytest.raises(RuntimeError, match=msg):
            paged_ops.paged_attention(*args)
    with pytest.raises(RuntimeError, match="workspace of"):
        paged_ops.paged_attention(q, k, k, t, n, workspace=z(64))
    with pytest.raises(RuntimeError, match="scale must be positive"):
        paged_ops.paged_attention(q, k, k, t, n, scale=-1.0)
    with pytest.raises(RuntimeError, match="q_starts must hold 4 rows"):
        paged_ops.prompt_attention(q, k, k, t, n, n)
    with pytest.raises(RuntimeError, match="prefix_len=33 positions exceed"):
        paged_ops.shared_prefix_attention(q, k, k, z(2, dtype=torch.int32), 33, t, n)
    i64 = torch.int64
    good = dict(qkv=z(3, 4 * 64), cos=z(8, 32, dtype=torch.float32), sin=z(8, 32, dtype=torch.float32),
                positions=z(3, dtype=i64), slots=z(3, dtype=i64), k_pages=k, v_pages=k, n_q_heads=2)
    for change, msg in ((dict(qkv=z(3, 200)), "qkv must be"), (dict(cos=z(8, 32)), "cos and sin"),
                        (dict(sin=z(8, 16, dtype=torch.float32)), "cos and sin"),
                        (dict(positions=z(2, dtype=i64)), "positions must hold 3"),
                        (dict(slots=z(3, dtype=torch.int32)), "slots must be"),
                        (dict(q_norm=z(64)), "given together"), (dict(q_norm=z(32), k_norm=z(64)), "q_norm must hold"),
                        (dict(cos=z(8, 33, dtype=torch.float32), sin=z(8, 33, dtype=torch.float32)), "rotary_dim")):
        with pytest.raises(RuntimeError, match=msg):
            paged_ops.rope_paged_append(**{**good, **change})
