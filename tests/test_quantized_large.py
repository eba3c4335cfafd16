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
