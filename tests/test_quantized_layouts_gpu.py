"""The 8-bit cache's operators on other layouts, streams and inputs than the
plain ones: strided pools, offsets past 32 bits, pages and slots out of range,
blocks that are not numbers in hidden places, large scales, waits that run out."""

from __future__ import annotations

import math

import pytest
import torch

from dequant_project_b200 import _native, paged_ops
from dequant_project_b200 import quantized_cache as qc
from test_quantized_cache_gpu import (CODES, TYPES, attend64, check_attention, clone, ints, largest_value, make_cache,
                                      query_rounding, reference, rows64, same_bits)

pytestmark = pytest.mark.gpu


def strided(cache):
    """The same cache in views: keys and values of one allocation each, heads
    outside pages, gaps between blocks' scales and open blocks."""
    n, hkv, page, d = cache.k.shape
    codes = torch.empty((hkv, n, 2, page, d + 16), dtype=torch.uint8, device=cache.k.device)
    k, v = (codes[:, :, i, :, :d].transpose(0, 1).view(cache.k.dtype) for i in (0, 1))
    scales = torch.empty((n, 2, hkv, cache.k_scale.shape[2] + 1), device=cache.k.device)
    ks, vs = (scales[:, i, :, :-1] for i in (0, 1))
    slots, _, block, _ = cache.k_open.shape
    opens = torch.empty((slots, 2, hkv, block * d + 8), dtype=cache.k_open.dtype, device=cache.k.device)
    ko, vo = (opens[:, i, :, :-8].unflatten(-1, (block, d)) for i in (0, 1))
    out = qc.QuantizedCache(k, v, ks, vs, ko, vo)
    for a, b in zip(out, cache):
        (a.view(torch.uint8) if a.element_size() == 1 else a).copy_(b.view(torch.uint8) if b.element_size() == 1 else b)
    return out


@pytest.mark.parametrize("d", [64, 128])
def test_strided_pools_and_queries(cuda_device, d):
    gen = torch.Generator(device=cuda_device).manual_seed(d)
    kl, hq, hkv = [300, 17, 64], 8, 2
    cache, table, slots = make_cache(gen, kl, hkv, d, 32, 16, torch.int8, torch.float16, cuda_device)
    view, lens = strided(cache), ints(kl, cuda_device)
    wide = torch.randn((90, hq, d + 8), generator=gen, device=cuda_device).half()
    q, starts = wide[:, :, :d], ints([0, 60, 70, 90], cuda_device)
    wide_table = torch.full((3, table.shape[1] + 3), -7, dtype=torch.int32, device=cuda_device)
    wide_table[:, :table.shape[1]] = table
    wt = wide_table[:, :table.shape[1]]
    n_pages = sum(-(-n // 32) for n in kl)
    assert torch.equal(qc.quantized_attention(q[:3], view, wt, slots, lens),
                       qc.quantized_attention(q[:3].contiguous(), cache, table, slots, lens))
    assert torch.equal(qc.quantized_prompt_attention(q, view, wt, slots, starts, lens, n_pages),
                       qc.quantized_prompt_attention(q.contiguous(), cache, table, slots, starts, lens, n_pages))
    for a, b in zip(qc.expanded_pages(view, wt, slots, lens, n_pages)[:2],
                    qc.expanded_pages(cache, table, slots, lens, n_pages)[:2]):
        assert torch.equal(a, b)
    cos, sin = paged_ops.rope_scaled_tables(d, 1e4, 512, cuda_device)
    qkv = torch.randn((90, (hq + 2 * hkv) * d), generator=gen, device=cuda_device).half()
    args = (qkv, cos, sin, torch.arange(90, device=cuda_device))
    assert torch.equal(qc.rope_quantized_append(*args, view, wt, slots, starts, lens, hq),
                       qc.rope_quantized_append(*args, cache, table, slots, starts, lens, hq))
    assert same_bits(view, cache)
    assert _native.device_status(cuda_device.index, reset=True) == 0


def test_offsets_past_32_bits(cuda_device):
    """Pages 2^29 bytes apart, open blocks 2^28 elements: codes past 2^32 bytes,
    open rows past 2^31 elements."""
    gen = torch.Generator(device=cuda_device).manual_seed(9)
    hkv, page, d, n = 2, 16, 128, 12
    cache, table, slots = make_cache(gen, [150], hkv, d, page, 16, torch.int8, torch.float16, cuda_device, extra=2)
    big = torch.empty(n << 29, dtype=torch.uint8, device=cuda_device)
    opens = torch.empty(n << 28, dtype=torch.float16, device=cuda_device)
    far = []
    move = torch.arange(n - 1, -1, -1, device=cuda_device)  # the far end holds page 0
    for which in (0, 1):
        codes = torch.as_strided(big, (n, hkv, page, d), (1 << 29, page * d, d, 1), which << 20).view(torch.int8)
        for i in range(n):
            codes[move[i]] = cache[which][i]
        scale = torch.empty((n, hkv, 1), device=cuda_device)
        scale[move] = cache[2 + which][:n]
        rows = torch.as_strided(opens, (n, hkv, 16, d), (1 << 28, 16 * d, d, 1), which << 20)
        rows[n - 1] = cache[4 + which][slots[0]]
        far.append((codes, scale, rows))
    there = qc.QuantizedCache(far[0][0], far[1][0], far[0][1], far[1][1], far[0][2], far[1][2])
    far_table = move[table.long().clamp(min=0)].int()
    far_slots, lens, starts = ints([n - 1], cuda_device), ints([150], cuda_device), ints([0, 20], cuda_device)
    q = torch.randn((20, 4, d), generator=gen, device=cuda_device).half()
    for f in (lambda c, t, s: qc.quantized_attention(q[:1], c, t, s, lens),
              lambda c, t, s: qc.quantized_prompt_attention(q, c, t, s, starts, lens, 10)):
        assert torch.equal(f(there, far_table, far_slots), f(cache, table, slots))
    cos, sin = paged_ops.rope_scaled_tables(d, 1e4, 256, cuda_device)
    qkv = torch.randn((20, 8 * d), generator=gen, device=cuda_device).half()
    pos = torch.arange(20, device=cuda_device)
    for c, t, s in ((there, far_table, far_slots), (cache, table, slots)):
        qc.rope_quantized_append(qkv, cos, sin, pos, c, t, s, starts, lens, 4)
    for which in (0, 1):
        assert torch.equal(rows64(there, which, far_table[0], n - 1, 150), rows64(cache, which, table[0], slots[0].long(), 150))


@pytest.mark.parametrize("codes", CODES, ids=str)
def test_large_and_small_scales_side_by_side(cuda_device, codes):
    """Values' scales from 2^-100 to 2^100 in one sequence, and keys' so that the
    large values' positions weigh little: sums keep what the softmax keeps."""
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    kl, hq, hkv, d = [1000, 70], 4, 2, 128
    cache, table, slots = make_cache(gen, kl, hkv, d, 32, 16, codes, torch.bfloat16, cuda_device)
    lens, q = ints(kl, cuda_device), torch.randn((2, hq, d), generator=gen, device=cuda_device).bfloat16()
    for power in (-100, 60, 100):
        c = clone(cache)
        pages = table[0, ::2].long()
        c.v_scale[pages] *= 2.0 ** power
        out = qc.quantized_attention(q, c, table, slots, lens)
        ref = reference(q, c, table, slots, kl, 1 / math.sqrt(d))
        for b in (0, 1):
            check_attention(out[b:b + 1], ref[b:b + 1], largest_value(c, table[b:b + 1], slots[b:b + 1], kl[b:b + 1]),
                            torch.bfloat16, query_rounding(q, c, table, slots, kl))
    # A huge block whose keys give it no weight at all changes nothing.
    c = clone(cache)
    last = table[0, 3].long()
    c.v_scale[last] *= 2.0 ** 100
    c.k_scale[last] = 0.5  # large scores of both signs
    q[0] = 0
    q[0, :, 0] = 40
    c.k.view(torch.uint8)[last, :, :, 0] = 0x81 if codes == torch.int8 else 0xfe  # all negative
    out = qc.quantized_attention(q, c, table, slots, lens)
    ref = reference(q, c, table, slots, kl, 1 / math.sqrt(d))
    seen = torch.cat([rows64(c, 1, table[0], slots[0].long(), 1000)[:96], rows64(c, 1, table[0], slots[0].long(), 1000)[128:]])
    check_attention(out[:1], ref[:1], float(seen.abs().max()), torch.bfloat16, query_rounding(q, c, table, slots, kl))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_hidden_blocks_that_are_not_numbers(cuda_device, dtype):
    """A block that a prompt's row does not see may have the scale NaN, or open
    rows that are not numbers, and does not matter to it; rows that see it give
    NaN."""
    gen = torch.Generator(device=cuda_device).manual_seed(6)
    n, hq, hkv, d = 300, 4, 2, 128
    cache, table, slots = make_cache(gen, [n], hkv, d, 32, 32, torch.int8, dtype, cuda_device)
    starts, lens = ints([0, n], cuda_device), ints([n], cuda_device)
    q = torch.randn((n, hq, d), generator=gen, device=cuda_device).to(dtype)
    want = qc.quantized_prompt_attention(q, cache, table, slots, starts, lens, 10)
    for which in (2, 3):
        bad = clone(cache)
        bad[which][table[0, 6].long()] = float("nan")   # positions 192 to 223
        out = qc.quantized_prompt_attention(q, bad, table, slots, starts, lens, 10)
        assert torch.equal(out[:192], want[:192]) and bool(out[192:].isnan().all())
    bad = clone(cache)
    bad.v_open[slots[0].long(), :, 5] = float("inf")  # position 293
    bad.k_open[slots[0].long(), :, 9] = float("nan")  # position 297
    out = qc.quantized_prompt_attention(q, bad, table, slots, starts, lens, 10)
    assert torch.equal(out[:293], want[:293]) and bool((out[293:297] == float("inf")).all())
    assert bool(out[297:].isnan().all())


def test_indexes_out_of_range_are_zeros_and_reported(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(7)
    kl, hq, hkv, d, page = [130, 70], 4, 2, 64, 32
    cache, table, slots = make_cache(gen, kl, hkv, d, page, 16, torch.int8, torch.float16, cuda_device)
    lens = ints(kl, cuda_device)
    q = torch.randn((2, hq, d), generator=gen, device=cuda_device).half()
    good = qc.quantized_attention(q, cache, table, slots, lens)
    pages = good.new_zeros(0)
    for bad in (-1, -(1 << 31), cache.k.shape[0], 1 << 30):
        t = table.clone()
        t[0, 1] = bad
        out = qc.quantized_attention(q, cache, t, slots, lens)
        assert _native.device_status(cuda_device.index, reset=True) == 2
        k, v = (rows64(cache, w, table[0], slots[0].long(), 130) for w in (0, 1))
        k[32:64] = v[32:64] = 0
        ref = attend64(q[:1], k, v, torch.tensor([130], device=q.device), 1 / math.sqrt(d))
        check_attention(out[:1], ref, float(v.abs().max()), torch.float16, query_rounding(q, cache, table, slots, kl))
        assert torch.equal(out[1], good[1])
        pages = qc.expanded_pages(cache, t, slots, lens, 8)[0]
        assert _native.device_status(cuda_device.index, reset=True) == 2
        assert bool((pages[1] == 0).all()) and bool((pages[0] != 0).any())
    for bad in (-1, cache.k_open.shape[0], 1 << 30):
        s = slots.clone()
        s[1] = bad
        out = qc.quantized_attention(q, cache, table, s, lens)
        assert _native.device_status(cuda_device.index, reset=True) == 2
        k, v = (rows64(cache, w, table[1], slots[1].long(), 70) for w in (0, 1))
        k[64:] = v[64:] = 0
        ref = attend64(q[1:], k, v, torch.tensor([70], device=q.device), 1 / math.sqrt(d))
        check_attention(out[1:], ref, float(v.abs().max()), torch.float16, query_rounding(q, cache, table, slots, kl))
        pages = qc.expanded_pages(cache, table, s, lens, 8)[0]
        assert _native.device_status(cuda_device.index, reset=True) == 2
        assert bool((pages[7] == 0).all())
    for n in (-3, 32 * table.shape[1] + 1, 1 << 30):
        out = qc.quantized_attention(q, cache, table, slots, ints([n, 70], cuda_device))
        assert _native.device_status(cuda_device.index, reset=True) & 2
        assert torch.equal(out[1], good[1])


def test_on_another_stream(cuda_device):
    """Calls go to torch's current stream: behind what it has in flight there."""
    gen = torch.Generator(device=cuda_device).manual_seed(8)
    cache, table, slots = make_cache(gen, [500], 2, 128, 32, 16, torch.int8, torch.float16, cuda_device)
    lens = ints([500], cuda_device)
    q = torch.randn((1, 8, 128), generator=gen, device=cuda_device).half()
    want = qc.quantized_attention(q, cache, table, slots, lens)
    late = torch.zeros_like(q)
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        late.copy_(q)
        out = qc.quantized_attention(late, cache, table, slots, lens)
    stream.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("bad,text", [
    (lambda c: c._replace(k=c.k.float()), "codes must be"),
    (lambda c: c._replace(v=c.v[:1]), "k and v must have one shape"),
    (lambda c: c._replace(k=c.k.cpu()), "k must be a CUDA tensor"),
    (lambda c: c._replace(v_open=c.v_open.cpu()), "v_open must be on"),
    (lambda c: c._replace(k_scale=c.k_scale.half()), "scales must be"),
    (lambda c: c._replace(k_scale=c.k_scale[:, :, :1].repeat(1, 1, 3), v_scale=c.v_scale[:, :, :1].repeat(1, 1, 3)),
     "do not hold"),
    (lambda c: c._replace(k_open=c.k_open.float(), v_open=c.v_open.float()), "open blocks must be float16"),
    (lambda c: c._replace(k_open=c.k_open.transpose(1, 2).contiguous().transpose(1, 2),
                          v_open=c.v_open.transpose(1, 2).contiguous().transpose(1, 2)), "last two dimensions"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_refused_caches(cuda_device, bad, text):
    cache = bad(qc.QuantizedCache.empty(4, 2, 32, 64, 2, device=cuda_device))
    q, one = torch.zeros((1, 4, 64), device=cuda_device).half(), ints([0], cuda_device)
    with pytest.raises(RuntimeError, match=text):
        qc.quantized_attention(q, cache, one[None], one, one)


def test_refused_arguments(cuda_device):
    cache = qc.QuantizedCache.empty(4, 2, 32, 64, 2, device=cuda_device)
    q, one = torch.zeros((1, 4, 64), device=cuda_device).half(), ints([0], cuda_device)
    for args, text in (((q.bfloat16(), one[None], one, one), "q must be"), ((q[:, :3], one[None], one, one), "head counts"),
                       ((q, one[None].long(), one, one), "block_table must be"), ((q, one[None], one.long(), one), "open_slots"),
                       ((q, one[None], one, ints([0, 0], cuda_device)), "kv_lens must hold 1 rows"),
                       ((q.cpu(), one[None], one, one), None)):
        if text is None:
            continue
        with pytest.raises(RuntimeError, match=text):
            qc.quantized_attention(args[0], cache, *args[1:])
    with pytest.raises(RuntimeError, match="workspace of"):
        qc.quantized_attention(q, cache, one[None], one, one, workspace=torch.zeros(16, dtype=torch.uint8, device=cuda_device))
    with pytest.raises(RuntimeError, match="scale must be positive"):
        qc.quantized_attention(q, cache, one[None], one, one, scale=0.0)
    with pytest.raises(RuntimeError, match="forward only"):
        qc.quantized_attention(q.requires_grad_(), cache, one[None], one, one)
    with torch.no_grad():
        assert bool((qc.quantized_attention(q, cache, one[None], one, one) == 0).all())


WAIT_NS = 2_000_000
COPIES = 128


def starved_call(q, cache, table, slots, lens, ws, out, mask):
    kv = _native.QuantizedKV(*(t.data_ptr() for t in cache), *cache.k.shape, cache.block, cache.k_open.shape[0],
                             *cache.k.stride()[:3], *cache.k_scale.stride()[:2], *cache.k_open.stride()[:2], 0, 0)
    _native.check(_native.lib().dqg_debug_quantized_starved(
        q.data_ptr(), q.stride(0), q.stride(1), q.shape[0], q.shape[1], kv, table.data_ptr(), table.shape[1],
        table.stride(0), slots.data_ptr(), lens.data_ptr(), 0.1, out.data_ptr(), ws.data_ptr(), ws.numel(), mask, WAIT_NS,
        torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("mask", [COPIES, 1, 4, 66], ids=["copies", "warp 0", "warp 2", "two warps"])
@pytest.mark.parametrize("kl,hq,hkv", [([700, 0, 33], 8, 2), ([40] * 300, 8, 2), ([500, 70], 40, 1)],
                         ids=["cut", "whole", "row blocks"])
def test_starved_kernels_give_up_and_report(cuda_device, kl, hq, hkv, mask):
    """Waits that run out end in an error status and NaN, not in a hang."""
    gen = torch.Generator(device=cuda_device).manual_seed(len(kl))
    cache, table, slots = make_cache(gen, kl, hkv, 128, 16, 16, torch.int8, torch.float16, cuda_device)
    lens = ints(kl, cuda_device)
    q = torch.randn((len(kl), hq, 128), generator=gen, device=cuda_device).half()
    size = q.numel()
    guarded = torch.full((3 * size,), 7.0, dtype=torch.float16, device=cuda_device)
    out = guarded[size:2 * size]
    ws = qc.quantized_attention_workspace(len(kl), hq, hkv, 128, cuda_device).fill_(255)
    torch.cuda.synchronize()
    _native.device_status(cuda_device.index, reset=True)
    starved_call(q, cache, table, slots, lens, ws, out, mask)
    torch.cuda.synchronize()  # returns: every wait gave up after WAIT_NS
    status = _native.device_status(cuda_device.index, reset=True)
    assert torch.isnan(out.float()).all()
    assert (guarded[:size] == 7.0).all() and (guarded[2 * size:] == 7.0).all()
    if mask == COPIES:
        assert status & 1, f"status {status:#x}: no wait reported giving up"
    # The context is still usable and the next call, on the same scratch, is right.
    want = qc.quantized_attention(q, cache, table, slots, lens)
    assert torch.isfinite(want).all()
    assert torch.equal(qc.quantized_attention(q, cache, table, slots, lens, workspace=ws), want)
    assert _native.device_status(cuda_device.index) == 0


def test_starved_rejects_bad_arguments(cuda_device):
    cache = qc.QuantizedCache.empty(4, 2, 32, 64, 2, device=cuda_device)
    q, one = torch.zeros((1, 4, 64), device=cuda_device).half(), ints([0], cuda_device)
    for mask in (0, 256):
        with pytest.raises(RuntimeError, match="starved must be"):
            starved_call(q, cache, one[None], one, one, q, q, mask)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("n,block", [(127, 32), (700, 64), (63, 64), (40, 16)])
def test_open_rows_beside_blocks_of_large_values(cuda_device, n, block, codes, dtype):
    """One channel's values are thousands of times the others', whose codes are
    zero beside it: what the other channels hold in the open rows is not lost. So
    check_attention's bound holds with a channel's own largest value (sums of zero
    codes are exact, those of int8 codes plus 128 too once as much is taken off)."""
    gen = torch.Generator(device=cuda_device).manual_seed(n)
    cache, table, slots = make_cache(gen, [n], 2, 128, 64, block, codes, dtype, cuda_device)
    cache.v.view(torch.uint8).fill_(0)
    cache.v.view(torch.uint8)[..., 5] = 0x7f if codes == torch.int8 else 0x7e
    cache.v_scale.fill_(60000 / qc.MOST[codes])
    opened = cache.v_open[int(slots[0]), :, :n % block]
    opened.copy_(1 + 0.2 * torch.randn(opened.shape, generator=gen, device=cuda_device))
    opened[..., 5] = 60000
    # (So many sequences, all of them this one, that no item is cut between the two.)
    many = 400
    q = torch.randn((many, 8, 128), generator=gen, device=cuda_device).to(dtype)
    out = qc.quantized_attention(q, cache, table.expand(many, -1).contiguous(), slots.expand(many).contiguous(),
                                 ints([n] * many, cuda_device))
    k, v = (rows64(cache, w, table[0], slots[0].long(), n) for w in (0, 1))
    ref = attend64(q, k, v, torch.full((many,), n, device=cuda_device), 1 / math.sqrt(128))
    channel = v.abs().amax(0).repeat_interleave(4, 0).clamp(min=1.0)
    check_attention(out.double() / channel, ref / channel, 1.0, dtype, query_rounding(q, cache, table, slots, [n]))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("d,g", [(128, 4), (64, 12)])
def test_a_query_channel_far_above_the_others(cuda_device, d, g, codes, dtype):
    """Queries with one value of 4000 among ordinary ones, over keys of zero
    there: nothing of the other channels is lost. Scores are fp32 sums of products
    with code + 128 at most, some ten in a row: e = scale s 2^-21 sum |q| (|code| +
    128)."""
    gen = torch.Generator(device=cuda_device).manual_seed(d)
    kl, hkv = [48, 63, 16, 7], 2
    cache, table, slots = make_cache(gen, kl, hkv, d, 16, 16, codes, dtype, cuda_device, spread=0.0)
    cache.k.view(torch.uint8)[..., 9] = 0
    cache.k_open[..., 9] = 0
    q = torch.randn((4, g * hkv, d), generator=gen, device=cuda_device).to(dtype)
    q[..., 9] = 4000
    out = qc.quantized_attention(q, cache, table, slots, ints(kl, cuda_device))
    ref = reference(q, cache, table, slots, kl, 1 / math.sqrt(d))
    most = 128 + qc.MOST[codes]
    step = float(cache.k_scale[table[0, 0].long()].max())
    e = 2.0 ** -21 * step * float(q.float().abs().sum(-1).max()) * most / math.sqrt(d)
    for b in range(4):
        one = table[b:b + 1], slots[b:b + 1], kl[b:b + 1]
        check_attention(out[b:b + 1], ref[b:b + 1], largest_value(cache, *one), dtype, e)


@pytest.mark.parametrize("power", [-110, -60, 60, 110, 118, 123])
@pytest.mark.parametrize("codes", CODES, ids=str)
def test_queries_of_any_size(cuda_device, codes, power):
    """bf16 queries times a power of two over keys (of blocks and open rows) by
    its inverse: the same scores, and the same result but for fp32 roundings."""
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    kl, d = [600, 45, 7], 128
    cache, table, slots = make_cache(gen, kl, 2, d, 32, 16, codes, torch.bfloat16, cuda_device)
    lens, q = ints(kl, cuda_device), torch.randn((3, 8, d), generator=gen, device=cuda_device).bfloat16()
    q[0, 1, 3] = q[1, 5, 100] = 13.0
    c = clone(cache)
    c.k_scale.mul_(2.0 ** -power)
    c.k_open.mul_(2.0 ** -power)
    out = qc.quantized_attention(q * 2.0 ** power, c, table, slots, lens)
    ref = reference(q, cache, table, slots, kl, 1 / math.sqrt(d))
    for b in range(3):
        one = table[b:b + 1], slots[b:b + 1], kl[b:b + 1]
        check_attention(out[b:b + 1], ref[b:b + 1], largest_value(cache, *one), torch.bfloat16,
                        query_rounding(q[b:b + 1], cache, *one))


def test_inputs_that_require_a_gradient_are_refused(cuda_device):
    """Codes in e4m3 as well, and a draw's parameters."""
    from dequant_project_b200.sampling import sample_tokens

    q, one, starts = torch.zeros((1, 4, 64), device=cuda_device).half(), ints([0], cuda_device), ints([0, 1], cuda_device)
    cos, sin = paged_ops.rope_scaled_tables(64, 1e4, 8, cuda_device)
    qkv = torch.zeros((1, 8 * 64), device=cuda_device).half()
    for which in range(6):
        cache = qc.QuantizedCache.empty(4, 2, 32, 64, 2, codes=torch.float8_e4m3fn, device=cuda_device)
        cache[which].requires_grad_()
        for call in (lambda: qc.quantized_attention(q, cache, one[None], one, one),
                     lambda: qc.quantized_prompt_attention(q, cache, one[None], one, starts, one, 1),
                     lambda: qc.expanded_pages(cache, one[None], one, one, 1),
                     lambda: qc.rope_quantized_append(qkv, cos, sin, one.long(), cache, one[None], one, starts,
                                                      one + 1, 4)):
            with pytest.raises(RuntimeError, match="forward only"):
                call()
    logits = torch.zeros((1, 4), device=cuda_device)
    args = dict(uniform=torch.zeros(1, device=cuda_device), temperature=torch.ones(1, device=cuda_device),
                top_p=torch.ones(1, device=cuda_device), min_p=torch.zeros(1, device=cuda_device))
    for name in args:
        with pytest.raises(RuntimeError, match="no gradient"):
            sample_tokens(logits, **{**args, name: args[name].clone().requires_grad_()})
    sample_tokens(logits, **args)


def test_queries_on_the_host_beside_a_cache_on_the_gpu_are_refused(cuda_device):
    cache = qc.QuantizedCache.empty(4, 2, 32, 64, 2, device=cuda_device)
    q, one, starts = torch.zeros((1, 4, 64)).half(), ints([0], cuda_device), ints([0, 1], cuda_device)
    cos, sin = paged_ops.rope_scaled_tables(64, 1e4, 8, cuda_device)
    for call, name in ((lambda: qc.quantized_attention(q, cache, one[None], one, one), "q"),
                       (lambda: qc.quantized_prompt_attention(q, cache, one[None], one, starts, one, 1), "q"),
                       (lambda: qc.rope_quantized_append(torch.zeros((1, 8 * 64)).half(), cos, sin, one.long(), cache,
                                                         one[None], one, starts, one + 1, 4), "qkv")):
        with pytest.raises(RuntimeError, match=f"^{name} must be float16 on cuda"):
            call()
    host = qc.QuantizedCache.empty(4, 2, 32, 64, 2, device="cpu")
    with pytest.raises(RuntimeError, match="k must be a CUDA tensor"):
        qc.quantized_attention(q.to(cuda_device), host, one[None], one, one)
