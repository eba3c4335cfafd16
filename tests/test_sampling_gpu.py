"""The draw of tokens on the GPU against the 64-bit restatement on the CPU.

The kernel's weights are exact to 2^-31 of themselves and rounded to 2^-45, their
sums exact; the restatement's sums are off by up to n 2^-53. So a running sum
differs by less than 2^-31 of itself and n 2^-45 of the largest weight (2^-27 for
n = 2^18), and a token can differ only where uniform * total, or top_p * total,
falls that near a border: for a random draw that is a chance of about n 2^-30.
With the fixed seeds here none does, so tokens are equal. Logprobs are formed in 64 bits and rounded
once: 2^-24 relative, and 2^-25 for what the sums are off.
"""

from __future__ import annotations

import pytest
import torch

from dequant_project_b200.sampling import sample_tokens

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]


def compare(logits, uniform, **params):
    tokens, logprobs = sample_tokens(logits, uniform, **params)
    cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in params.items()}
    want, want_lp = sample_tokens(logits.cpu(), uniform.cpu(), **cpu)
    assert torch.equal(tokens.cpu(), want), (tokens.cpu()[tokens.cpu() != want], want[tokens.cpu() != want])
    lp = logprobs.cpu()
    assert torch.equal(lp.isnan(), want_lp.isnan())
    ok = (lp - want_lp).abs() <= 2.0 ** -23 * want_lp.abs() + 2.0 ** -25
    assert bool((ok | lp.isnan()).all())
    again = sample_tokens(logits, uniform, **params)
    assert torch.equal(again[0], tokens) and torch.equal(again[1].view(torch.int32), logprobs.view(torch.int32))
    return tokens.cpu()


def rows_of(gen, rows, vocab, dtype, device, spread=3.0):
    logits = (spread * torch.randn((rows, vocab), generator=gen, device=device)).to(dtype)
    return logits, torch.rand(rows, generator=gen, device=device).clamp(max=1 - 2.0 ** -24)


PARAMS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.0),
          dict(min_p=0.05), dict(top_k=40, top_p=0.95, min_p=0.02, temperature=1.3), dict(temperature=0.0),
          dict(top_k=7, top_p=0.5), dict(top_p=0.999, temperature=2.0), dict(min_p=1.0), dict(top_k=10 ** 9, top_p=2.0)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("params", PARAMS, ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (4, 33), (2, 1000), (7, 4099), (3, 32000)])
def test_draws(cuda_device, rows, vocab, params, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(rows * vocab)
    compare(*rows_of(gen, rows, vocab, dtype, cuda_device), **params)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab", [(2, 128256), (1, 262144), (300, 500), (160, 32000), (33, 50257)])
def test_many_rows_and_wide_ones(cuda_device, rows, vocab, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(vocab)
    logits, uniform = rows_of(gen, rows, vocab, dtype, cuda_device)

    def each(lo, hi):
        return lo + (hi - lo) * torch.rand(rows, generator=gen, device=cuda_device)

    heat = torch.where(each(0, 1) < 0.2, 0.0, each(0.2, 1.5))
    compare(logits, uniform, temperature=heat, top_k=each(-50, 300).int(), top_p=each(0.3, 1.1), min_p=each(-0.1, 0.1))


def test_wide_rows_without_any_filter(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    for spread in (0.01, 1.0, 10.0):
        compare(*rows_of(gen, 40, 128256, torch.float32, cuda_device, spread))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_ties_are_kept_from_the_lowest_index(cuda_device, dtype):
    """Equal logits: k of them are the first k; top_p of n equal ones the first
    ceil(p n). (Weights of 1 add exactly on both sides.)"""
    n = 5000
    logits = torch.zeros((6, n), device=cuda_device, dtype=dtype)
    logits[1:, ::2] = -0.0
    uniform = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999, 1 - 2.0 ** -24], device=cuda_device)
    assert compare(logits, uniform).tolist() == [int(float(u) * n) for u in uniform.cpu()]
    assert compare(logits, uniform, top_k=8).tolist() == [0, 2, 4, 6, 7, 7]
    assert compare(logits, uniform, top_p=0.5).tolist() == [int(float(u) * 2500) for u in uniform.cpu()]
    logits[:, 4000:] = 1.0
    assert compare(logits, uniform, top_k=1004).max() < n
    tokens = compare(logits, uniform, top_k=1001, temperature=1e30)
    assert tokens[0] == 0 and tokens[1:].min() >= 4000
    few = torch.randint(-3, 4, (50, n), device=cuda_device).to(dtype)
    u = torch.rand(50, device=cuda_device)
    for params in (dict(top_k=100), dict(top_p=0.7), dict(top_k=2000, top_p=0.3), dict(min_p=0.1, top_p=0.8)):
        compare(few, u, **params)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_masked_rows_infinities_and_nan(cuda_device, dtype):
    inf, nan = float("inf"), float("nan")
    rows = torch.full((8, 3001), -inf)
    rows[1, 1234] = -5.0
    rows[2] = nan
    rows[3, [7, 9, 2000]] = inf
    rows[4] = 0.0
    rows[4, 5] = nan
    rows[5, 3000] = torch.finfo(dtype).min
    rows[6] = torch.finfo(dtype).min
    rows[7, ::3] = 1.0
    logits = rows.to(dtype).to(cuda_device)
    for u in (0.0, 0.4, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, nan):
        uniform = torch.full((8,), u, device=cuda_device)
        for params in (dict(), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.5), dict(temperature=0.0)):
            tokens, logprobs = (t.cpu() for t in sample_tokens(logits, uniform, **params))
            if 0.0 <= u < 1.0:
                compare(logits, uniform, **params)
            assert tokens[0] == -1 and tokens[2] == -1 and logprobs[0].isnan() and logprobs[2].isnan()
            assert tokens[1] == 1234 and logprobs[1] == 0.0
            assert int(tokens[3]) in (7, 9, 2000) and tokens[4] != 5 and tokens[5] == 3000 and tokens[7] % 3 == 0
            assert bool((tokens[[4, 6, 7]] >= 0).all())


def test_parameters_out_of_range_and_of_each_row(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    logits, uniform = rows_of(gen, 4, 777, torch.float32, cuda_device)
    nan, inf = float("nan"), float("inf")
    best = logits.argmax(1).cpu()
    for t in (0.0, -1.0, nan):
        assert torch.equal(sample_tokens(logits, uniform, temperature=t)[0].cpu(), best)
    assert torch.equal(sample_tokens(logits, uniform, temperature=1e-30)[0].cpu(), best)
    assert torch.equal(sample_tokens(logits, uniform, top_p=-1.0)[0].cpu(), best)
    assert torch.equal(sample_tokens(logits, uniform, min_p=5.0)[0].cpu(), best)
    plain = sample_tokens(logits, uniform)[0]
    for params in (dict(top_p=nan), dict(min_p=nan), dict(top_k=-3), dict(top_p=inf), dict(min_p=-inf)):
        assert torch.equal(sample_tokens(logits, uniform, **params)[0], plain)
    flat = sample_tokens(logits, uniform, temperature=inf)[0].cpu()
    assert flat.tolist() == [int(float(u) * 777) for u in uniform.cpu().double()]
    k = torch.tensor([1, 0, 5, 700], dtype=torch.int32, device=cuda_device)
    both = sample_tokens(logits, uniform, top_k=k)[0]
    for r in range(4):
        assert both[r] == sample_tokens(logits[r:r + 1], uniform[r:r + 1], top_k=int(k[r]))[0][0]


def test_rows_apart_and_unaligned(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    for dtype in TYPES:
        wide = torch.randn((9, 1003), generator=gen, device=cuda_device).to(dtype)
        uniform = torch.rand(9, generator=gen, device=cuda_device)
        for lo, hi in ((0, 1003), (1, 1000), (3, 998), (8, 9)):
            view = wide[:, lo:hi]
            assert torch.equal(sample_tokens(view, uniform, top_p=0.9)[0],
                               sample_tokens(view.contiguous(), uniform, top_p=0.9)[0])


def test_captured_draws_on_another_stream(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    logits, uniform = rows_of(gen, 5, 32000, torch.float16, cuda_device)
    heat = torch.full((5,), 0.8, device=cuda_device)
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        sample_tokens(logits, uniform, temperature=heat, top_p=0.9)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        tokens, _ = sample_tokens(logits, uniform, temperature=heat, top_p=0.9)
    for _ in range(3):
        logits.copy_(torch.randn(logits.shape, generator=gen, device=cuda_device))
        uniform.copy_(torch.rand(5, generator=gen, device=cuda_device))
        heat.copy_(heat * 1.1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, sample_tokens(logits, uniform, temperature=heat, top_p=0.9)[0])


def test_refusals(cuda_device):
    x, u = torch.randn((2, 100), device=cuda_device), torch.rand(2, device=cuda_device)
    for args, params, text in (
            ((x.double(), u), {}, "logits must be"), ((x[0], u), {}, "rows, vocab"), ((x.t(), u), {}, "contiguous rows"),
            ((x, u.double()), {}, "uniform must be"), ((x, u[:1]), {}, "uniform must be"), ((x, u.cpu()), {}, "uniform"),
            ((x, u), dict(temperature=u.double()), "temperature must be"), ((x, u), dict(top_k=u), "top_k must be"),
            ((x, u), dict(top_p=torch.rand(3, device=cuda_device)), "top_p must be"),
            ((x.expand(2, 100).requires_grad_(), u), {}, "no gradient"),
            ((torch.zeros((1, 2 ** 18 + 1), device=cuda_device), u[:1]), {}, "vocab must be"),
            ((torch.zeros((2, 0), device=cuda_device), u), {}, "vocab must be")):
        with pytest.raises(RuntimeError, match=text):
            sample_tokens(*args, **params)
    tokens, logprobs = sample_tokens(x[:0], u[:0])
    assert tokens.shape == (0,) and logprobs.shape == (0,)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_min_p_above_one_keeps_the_first_of_equal_logits(cuda_device, dtype):
    logits = torch.zeros((5, 3000), dtype=dtype, device=cuda_device)
    logits[1, 70:] = 2.0
    logits[2, [5, 2999]] = float("inf")
    logits[3] = float("nan")
    logits[4, 2000:] = -1.0
    for u in (0.0, 0.5, 0.99):
        uniform = torch.full((5,), u, device=cuda_device)
        for params in (dict(min_p=5.0), dict(min_p=1.0 + 2.0 ** -23, temperature=0.7), dict(min_p=2.0, top_k=100),
                       dict(min_p=float("inf"), top_p=0.5)):
            assert compare(logits, uniform, **params).tolist() == [0, 70, 5, -1, 0]
        assert compare(logits, uniform, min_p=1.0)[4] == int(u * 2000)
    each = torch.tensor([5.0, 1.0, 0.5, 2.0, 3.0], device=cuda_device)
    assert compare(logits, torch.full((5,), 0.99, device=cuda_device), min_p=each)[0] == 0
