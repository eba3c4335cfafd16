"""The 8-bit cache's operators and the token draw on CPU tensors: the formulas
that the GPU tests compare with, and what the calls refuse."""

from __future__ import annotations

import math

import pytest
import torch

from dequant_project_b200 import paged_ops
from dequant_project_b200 import quantized_cache as qc
from dequant_project_b200.sampling import sample_tokens


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("block,page", [(16, 16), (32, 64), (64, 128)])
def test_prompt_cut_in_any_way_gives_the_same_cache_and_attention(block, page, codes):
    gen = torch.Generator().manual_seed(block)
    n, hq, hkv, d = 150, 4, 2, 64
    qkv = torch.randn((n, (hq + 2 * hkv) * d), generator=gen).half()
    cos, sin = paged_ops.rope_scaled_tables(d, 1e4, 256, "cpu")
    table = torch.randperm(-(-n // page), generator=gen).int()[None]
    caches, queries = [], []
    for cuts in ([n], [1] * n, [5, 11, 16, 32, 1, 63, 22]):
        cache = qc.QuantizedCache.empty(-(-n // page), hkv, page, d, 2, block=block, codes=codes, device="cpu")
        at, q = 0, []
        for c in cuts:
            q.append(qc.rope_quantized_append(qkv[at:at + c], cos, sin, torch.arange(at, at + c), cache, table, ints(1),
                                              ints(0, c), ints(at + c), hq))
            at += c
        for x in cache[4:]:
            x[1, :, n % block:] = 0
        caches.append(cache)
        queries.append(torch.cat(q))
    for other, q in zip(caches[1:], queries[1:]):
        assert torch.equal(q, queries[0])
        for x, y in zip(other, caches[0]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    # Against the 16-bit cache: a code is off by half a step, and a step is the
    # block's largest value / 127 (int8) or 2^-3 of the value (e4m3).
    k, v = (torch.zeros((-(-n // page), hkv, page, d), dtype=torch.float16) for _ in range(2))
    slots = table[0].long()[torch.arange(n) // page] * page + torch.arange(n) % page
    paged_ops.rope_paged_append(qkv, cos, sin, torch.arange(n), slots, k, v, hq)
    ek, ev, et = qc.expanded_pages(caches[0], table, ints(1), ints(n), -(-n // page))
    for a, b in ((k, ek), (v, ev)):
        a, b = a[table[0].long()], b[et[0].long()]
        rel = 2.0 ** -4 if codes == torch.float8_e4m3fn else 0.0
        step = float(a.abs().max()) / (127 if codes == torch.int8 else 448 * 2 ** 9)
        assert bool(((a - b).float().abs() <= (rel + 2.0 ** -10) * a.float().abs() + 0.51 * step).all())
    out = qc.quantized_prompt_attention(queries[0], caches[0], table, ints(1), ints(0, n), ints(n), -(-n // page))
    want = paged_ops.prompt_attention(queries[0], ek, ev, et, ints(0, n), ints(n))
    last = qc.quantized_attention(queries[0][-1:], caches[0], table, ints(1), ints(n))
    # (The expanded pages' values are rounded to fp16 once more: 2^-11 of each, and of the scores' keys.)
    e = 2.0 ** -11 * float(queries[0].float().norm(dim=-1).max() * ek.float().norm(dim=-1).max()) / math.sqrt(d)
    assert float((out - want).abs().max()) <= (2.0 ** -10 + math.expm1(2 * e)) * float(ev.abs().max())
    assert float((last[0] - out[-1]).abs().max()) <= 2.0 ** -9 * float(ev.abs().max())


def test_a_block_with_a_value_that_is_not_finite_reads_as_nan():
    for codes in (torch.int8, torch.float8_e4m3fn):
        x = torch.ones((3, 16, 64)).half()
        x[1, 5, 6] = float("inf")
        x[2] = 0
        c, s = qc.quantize_block(x, codes)
        assert s[0] == 1 / qc.MOST[codes] and s[1].isnan() and s[2] == qc.LEAST_SCALE
        assert bool((c[1].float() == 0).all() and (c[2].float() == 0).all())


def test_refusals():
    for bad in (dict(block=8), dict(block=64), dict(codes=torch.float16)):
        with pytest.raises(ValueError):
            qc.QuantizedCache.empty(2, 1, 32, 64, 1, device="cpu", **bad)
    cache = qc.QuantizedCache.empty(2, 1, 32, 64, 1, device="cpu")
    q = torch.zeros((1, 1, 64)).half().requires_grad_()
    with pytest.raises(RuntimeError, match="forward only"):
        qc.quantized_attention(q, cache, ints(0)[None], ints(0), ints(1))
    with pytest.raises(RuntimeError, match="no gradient"):
        sample_tokens(torch.zeros((1, 4), requires_grad=True), torch.zeros(1))


def test_draws_by_hand():
    """Logits 0, ln 2, ln 4, ln 1: weights 1, 2, 4, 1 of 8."""
    logits = torch.tensor([[0.0, math.log(2), math.log(4), 0.0]], dtype=torch.float64).float()

    def token(u, **params):
        t, lp = sample_tokens(logits, torch.tensor([u]), **params)
        return int(t), float(lp.exp())

    assert [token(u)[0] for u in (0.0, 0.12, 0.13, 0.37, 0.38, 0.87, 0.88, 0.9999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert token(0.5)[1] == pytest.approx(0.5)
    assert token(0.99, top_k=3)[0] == 2 and token(0.0, top_k=3)[0] == 0       # of the two 1s the first
    assert token(0.0, top_k=2) == (1, pytest.approx(1 / 3))
    assert token(0.0, top_p=0.5)[0] == 2                                      # 4 of 8 reach it alone
    assert token(0.0, top_p=0.51)[0] == 1 and token(0.0, top_p=0.76)[0] == 0
    assert token(0.99, top_p=0.76)[0] == 2                                    # 4 + 2 + the first 1
    assert token(0.0, top_k=2, top_p=0.66)[0] == 2 and token(0.0, top_k=2, top_p=0.67)[0] == 1
    assert token(0.0, min_p=0.3)[0] == 1 and token(0.0, min_p=0.2)[0] == 0
    assert token(0.9, temperature=0.0) == (2, 1.0) and token(0.9, top_p=0.0) == (2, 1.0)
    assert token(0.32, temperature=0.5)[0] == 2                               # weights 1, 4, 16, 1 of 22
    assert token(0.22, temperature=0.5)[0] == 1


@pytest.mark.parametrize("name", ["uniform", "temperature", "top_p", "min_p"])
def test_draws_refuse_parameters_that_require_a_gradient(name):
    args = dict(uniform=torch.full((2,), 0.5), temperature=torch.ones(2), top_p=torch.ones(2), min_p=torch.zeros(2))
    args[name].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        sample_tokens(torch.zeros((2, 4)), **args)
    with torch.no_grad():
        assert sample_tokens(torch.zeros((2, 4)), **args)[0].tolist() == [2, 2]
