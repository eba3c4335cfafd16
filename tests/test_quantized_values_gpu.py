"""Values of an 8-bit cache in prompt attention: a block's scale as a power of
two, which the 16-bit values take exactly, times a factor in [1, 2), which goes
to the softmax's weights. On the GPU, against a 64-bit restatement.

The only roundings to 16 bits are the output's and each weight's: with u the
type's unit roundoff |out - ref| <= u |ref| + (u + 2^-13) max|v|, the 2^-13 for
exponentials and fp32 sums. fp16 values below its normal numbers are off by up to
2^-25 before the factor: 2^-24 more where a scale is that small.
"""

from __future__ import annotations

import math

import pytest
import torch

from dequant_project_b200 import _native
from dequant_project_b200 import quantized_cache as qc
from test_quantized_cache_gpu import CODES, TYPES, U, attend64, ints, make_cache, rows64

pytestmark = pytest.mark.gpu


def case(device, seed, n, hq, hkv, d, page, block, codes, dtype, n_q):
    gen = torch.Generator(device=device).manual_seed(seed)
    cache, table, slots = make_cache(gen, [n], hkv, d, page, block, codes, dtype, device)
    q = torch.randn((n_q, hq, d), generator=gen, device=device).to(dtype)
    return gen, cache, table, slots, q


def attend(q, cache, table, slots, n, **kw):
    device = q.device
    return qc.quantized_prompt_attention(q, cache, table, slots, ints([0, q.shape[0]], device), ints([n], device),
                                         -(-n // cache.page_size), **kw)


def reference(q, cache, table, slots, n, scale=None):
    k, v = (rows64(cache, w, table[0], slots[0].long(), n) for w in (0, 1))
    ends = n - q.shape[0] + torch.arange(q.shape[0], device=q.device) + 1
    return attend64(q, k, v, ends, 1 / math.sqrt(q.shape[2]) if scale is None else scale), v


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("n,n_q,hq,hkv,d,page,block", [
    (1000, 300, 8, 2, 128, 16, 16), (640, 640, 4, 4, 64, 32, 32), (333, 1, 16, 1, 128, 256, 64), (129, 129, 28, 4, 64, 64, 16),
])
def test_values_are_rounded_nowhere(cuda_device, n, n_q, hq, hkv, d, page, block, codes, dtype):
    gen, cache, table, slots, q = case(cuda_device, n, n, hq, hkv, d, page, block, codes, dtype, n_q)
    # Factors over all of [1, 2), its ends among them.
    s = cache.v_scale
    factor = 1 + torch.rand(s.shape, generator=gen, device=cuda_device)
    factor.view(-1)[::5] = 1.0
    factor.view(-1)[1::5] = 2 - 2.0 ** -23
    s.copy_(torch.where(s.isnan(), s, factor * 2.0 ** torch.randint(-9, -4, s.shape, generator=gen, device=cuda_device)))
    out = attend(q, cache, table, slots, n)
    ref, v = reference(q, cache, table, slots, n)
    u = U[dtype]
    lim = u * ref.abs() + (u + 2.0 ** -13) * float(v.abs().max()) + 1e-7
    assert bool(((out.double() - ref).abs() <= lim).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("codes", CODES, ids=str)
def test_scales_of_any_size(cuda_device, codes, dtype):
    """Blocks of zeros (the least scale there is, and zero), of very small and
    of large values, beside one another; and one that is not a number, which the
    rows before it do not see."""
    n, block = 400, 16
    gen, cache, table, slots, q = case(cuda_device, 5, n, 8, 2, 128, 16, block, codes, dtype, n)
    pages = table[0].long()
    cache.v.view(torch.uint8)[pages[2]] = 0
    cache.v_scale[pages[2]] = 2.0 ** -126
    cache.v_scale[pages[3]] = 0.0
    cache.v_scale[pages[4]] = 1.75 * 2.0 ** -27
    cache.v_scale[pages[5]] = 1.25 * 2.0 ** -126
    cache.v_scale[pages[6]] = 1.9 * (64.0 if codes == torch.int8 else 16.0)
    out = attend(q, cache, table, slots, n)
    ref, v = reference(q, cache, table, slots, n)
    u = U[dtype]
    # Rows see values of very different sizes: of those up to each row's end.
    top = v.abs().amax((1, 2)).cummax(0).values[:, None, None]
    lim = u * ref.abs() + (u + 2.0 ** -13) * top + 2.0 ** -24
    assert bool(((out.double() - ref).abs() <= lim).all())
    cache.v_scale[pages[20]] = float("nan")
    again = attend(q, cache, table, slots, n)
    first = 20 * block
    assert torch.equal(again[:first], out[:first]) and bool(again[first:].isnan().all())
    assert _native.device_status(cuda_device.index, reset=True) == 0


@pytest.mark.parametrize("scale", [1e-36, 1e-20, 30.0, 1e4])
def test_softmax_scales_of_any_size(cuda_device, scale):
    """A factor's logarithm is divided by the softmax's scale. Where that is
    below 1e-30 values are rounded instead: u of themselves. Large scales leave
    what the scores' own roundings, of their fp32 sums, make of the weights: e =
    scale 2^-18 sum |q||k| moves an output by expm1(2 e) max|v| (of those that
    hold, e < 0.1, up to 30 here; beyond, no row may be but a mean of its values)."""
    n = 300
    _, cache, table, slots, q = case(cuda_device, 7, n, 4, 2, 64, 32, 16, torch.int8, torch.float16, 100)
    q = q * 0.125
    out = attend(q, cache, table, slots, n, scale=scale)
    ref, v = reference(q, cache, table, slots, n, scale)
    u, most = U[torch.float16], float(v.abs().max())
    assert bool(out.isfinite().all()) and float(out.abs().max()) <= (1 + 2 * u) * most
    if scale <= 30:
        k, _ = (rows64(cache, w, table[0], slots[0].long(), n) for w in (0, 1))
        e = scale * 2.0 ** -18 * float(q.double().abs().sum(-1).max()) * float(k.abs().max())
        lim = u * ref.abs() + (2 * u + 2.0 ** -13 + math.expm1(2 * e)) * most + 1e-7
        assert bool(((out.double() - ref).abs() <= lim).all())

