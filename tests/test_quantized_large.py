"""Blocks of an 8-bit cache whose values are near the largest that bf16 has: a
code is formed as a quotient of L times the value, which fp32 cannot hold.

A scale is fp32(max|x| / L) exactly, and a code off by at most half a step (1 for
int8, 2^-3 of the power of two at or below the quotient for e4m3) and 2^-22 of the
quotient for fp32 roundings (the scale's among them)."""

from __future__ import annotations

import pytest
import torch

from dequant_project_b200 import quantized_cache as qc

CODES = [torch.int8, torch.float8_e4m3fn]
LARGE = [3.3895313892515355e38, 1e37, 2.0 ** 113, 7e29]  # bf16's largest first


def large_blocks(device):
    """A bf16 batch of one token block each, whose largest magnitudes are LARGE."""
    gen = torch.Generator().manual_seed(3)
    x = 2 * torch.rand((len(LARGE), 16, 64), generator=gen) - 1
    x[:, 0, 0] = torch.tensor([1.0, -1.0, 1.0, -1.0])
    return (x.double() * torch.tensor(LARGE).double()[:, None, None]).to(torch.bfloat16).to(device)


def check_large(codes, scale, x):
    x = x.cpu().double()
    most = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}[codes.dtype]
    assert torch.equal(scale.cpu(), (x.abs().amax((1, 2)) / most).float())
    y = x / scale.cpu().double()[:, None, None]
    got = codes.cpu().float().double()
    if codes.dtype == torch.int8:
        step = torch.ones_like(y)
    else:
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    assert bool(((got - y).abs() <= step / 2 + 2.0 ** -22 * y.abs()).all())


@pytest.mark.parametrize("codes", CODES, ids=str)
def test_restatement(codes):
    x = large_blocks("cpu")
    check_large(*qc.quantize_block(x, codes), x)


@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
def test_kernel(cuda_device, codes):
    x = large_blocks(cuda_device)
    n, d = len(LARGE), 64

    def ints(values):
        return torch.tensor(list(values), dtype=torch.int32, device=cuda_device)

    cache = qc.QuantizedCache.empty(n, 1, 16, d, n, codes=codes, dtype=torch.bfloat16, device=cuda_device)
    qkv = torch.zeros((16 * n, 3 * d), dtype=torch.bfloat16, device=cuda_device)
    qkv[:, 2 * d:] = x.reshape(-1, d)
    at = torch.zeros(16 * n, dtype=torch.int64, device=cuda_device)
    cos, sin = torch.ones((1, d // 2), device=cuda_device), torch.zeros((1, d // 2), device=cuda_device)
    table = torch.arange(n, device=cuda_device, dtype=torch.int32)[:, None]
    qc.rope_quantized_append(qkv, cos, sin, at, cache, table, ints(range(n)),
                             ints(range(0, 16 * n + 1, 16)), ints([16] * n), 1)
    check_large(cache.v[:, 0], cache.v_scale[:, 0, 0], x)


def appended(device, n, g, page, block, most, codes, d=64, hkv=2):
    """A bf16 sequence of n positions whose values are up to ``most``, appended:
    the queries, the cache and what goes with it, and its 64-bit keys and values."""
    from test_quantized_cache_gpu import ints, rows64

    gen = torch.Generator(device=device).manual_seed(n)
    cache = qc.QuantizedCache.empty(-(-n // page), hkv, page, d, 1, block=block, codes=codes, dtype=torch.bfloat16,
                                    device=device)
    qkv = torch.randn((n, (g + 2) * hkv * d), generator=gen, device=device)
    qkv[:, -hkv * d:].uniform_(-1, 1, generator=gen).mul_(most)
    qkv[n // 2, -hkv * d:] = -most
    cos, sin = torch.ones((1, d // 2), device=device), torch.zeros((1, d // 2), device=device)
    table = torch.randperm(-(-n // page), generator=gen, device=device).int()[None]
    slot = ints([0], device)
    q = qc.rope_quantized_append(qkv.bfloat16(), cos, sin, torch.zeros(n, dtype=torch.int64, device=device), cache,
                                 table, slot, ints([0, n], device), ints([n], device), g * hkv)
    return q, cache, table, slot, *(rows64(cache, w, table[0], 0, n) for w in (0, 1))


SIZES = [(37, 1, 16, 16), (9, 4, 64, 64), (64, 8, 64, 64), (3000, 12, 128, 32)]  # n, heads a KV head, page, block


@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("most", LARGE + [1e34, 1e-30])
@pytest.mark.parametrize("n,g,page,block", SIZES)
def test_decode_over_large_values(cuda_device, n, g, page, block, most, codes):
    """|out - ref| <= u |ref| + (u + 2^-13) max|v| as for ordinary values (and, for
    queries beside int8 codes, what test_quantized_cache_gpu.py allows), for a
    sequence cut into pieces and for many that are not."""
    from test_quantized_cache_gpu import attend64, check_attention, ints, query_rounding

    q, cache, table, slot, k, v = appended(cuda_device, n, g, page, block, most, codes)
    unit = float(v.abs().max())
    for rows in (1, min(n, 400)):
        last = q[-rows:].contiguous()
        out = qc.quantized_attention(last, cache, table.expand(rows, -1).contiguous(), slot.expand(rows).contiguous(),
                                     ints([n] * rows, cuda_device))
        ref = attend64(last, k, v, torch.full((rows,), n, device=cuda_device), 0.125)
        check_attention(out.double() / unit, ref / unit, 1.0, torch.bfloat16,
                        query_rounding(last, cache, table, slot, [n]))


@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
def test_values_of_zero_scales_and_low_scores(cuda_device, codes):
    """Blocks whose values' scales are zero read as zeros, whatever the scores are."""
    from test_quantized_cache_gpu import ints

    q, cache, table, slot, _, _ = appended(cuda_device, 64, 2, 16, 16, 1.0, codes)
    cache.v_scale.zero_()
    cache.k_scale.fill_(1.0)
    cache.k.view(torch.uint8).fill_(0x81 if codes == torch.int8 else 0xfe)  # the most negative
    out = qc.quantized_attention(torch.full_like(q[:1], 100.0), cache, table, slot, ints([64], cuda_device))
    assert bool((out == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("most", LARGE + [1e34, 1e-30])
@pytest.mark.parametrize("n,g,page,block", SIZES)
def test_prompts_over_large_values(cuda_device, n, g, page, block, most, codes):
    """|out - ref| <= u |ref| + (u + 2^-13) max|v|, as for ordinary values."""
    from test_quantized_cache_gpu import attend64, check_attention, ints

    q, cache, table, slot, k, v = appended(cuda_device, n, g, page, block, most, codes)
    unit, rows = float(v.abs().max()), min(n, 200)
    ends = n - rows + 1 + torch.arange(rows, device=cuda_device)
    last = q[-rows:].contiguous()
    out = qc.quantized_prompt_attention(last, cache, table, slot, ints([0, rows], cuda_device), ints([n], cuda_device),
                                        -(-n // page))
    check_attention(out.double() / unit, attend64(last, k, v, ends, 0.125) / unit, 1.0, torch.bfloat16)
