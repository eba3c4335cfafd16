"""Serving with a cache held in 8 bits on the GPU: a ``PagedDecoder`` with one
against a 16-bit one. The first layer's keys and values depend on the tokens
alone: its codes are checked against the 16-bit cache's values (a scale
exactly, a code to half a step; prompts above eight rows of either decoder go
through the same products). Logits: see test_quantized_decoder.py."""

from __future__ import annotations

import pytest
import torch

from decoder_reference import max_rel_err
from dequant_project_b200 import _native
from dequant_project_b200 import quantized_cache as qc
from dequant_project_b200.decoder import TPDecoder
from dequant_project_b200.paged_decoder import PagedDecoder
from test_paged_decoder_gpu import CFG, QCFG
from test_quantized_cache_gpu import check_codes

pytestmark = pytest.mark.gpu

BOUND = {torch.int8: 0.05, torch.float8_e4m3fn: 0.25}


@pytest.mark.parametrize("codes", list(BOUND), ids=str)
@pytest.mark.parametrize("prefix", [0, 64])
def test_against_the_16_bit_cache(cuda_device, codes, prefix):
    dec = TPDecoder(CFG, QCFG, seed=3, device=cuda_device, batch=4, kv_len=0)
    gen = torch.Generator().manual_seed(prefix)
    toks = [torch.randint(0, CFG.vocab, (n,), generator=gen) for n in (1, 16, 33, 90)]
    head = torch.randint(0, CFG.vocab, (max(prefix, 1),), generator=gen)
    more = torch.randint(0, CFG.vocab, (4, 20), generator=gen)
    both, results = [], []
    for c in (None, codes):
        serve = PagedDecoder(dec, n_pages=64, page_size=32, max_positions=256, codes=c, block=32)
        if prefix:
            serve.set_prefix(head)
        ids, logits = serve.add(toks)
        results.append([logits] + [serve.step(ids, more[:, i]) for i in range(20)])
        both.append(serve)
    assert _native.device_status(cuda_device.index, reset=True) == 0
    for a, b in zip(*results):
        assert max_rel_err(b.float(), a.float()) < BOUND[codes]
    plain, serve = both
    cache = serve.cache[0]
    for i in ids:
        pages, n = plain.prefix_pages + plain.seqs[i]["pages"], prefix + plain.seqs[i]["len"]
        assert serve.prefix_pages + serve.seqs[i]["pages"] == pages
        for page, base in zip(pages, range(0, n, 32)):
            for which, x in ((0, plain.k[0][page]), (1, plain.v[0][page])):
                if base + 32 <= n:
                    check_codes(cache[which][page], cache[2 + which][page, :, 0], x)
                else:
                    assert torch.equal(cache[4 + which][serve.seqs[i]["open"], :, :n - base], x[:, :n - base])


def test_generate_draws_what_its_generator_says(cuda_device):
    dec = TPDecoder(CFG, QCFG, seed=3, device=cuda_device, batch=4, kv_len=0)
    serve = PagedDecoder(dec, n_pages=64, page_size=16, max_positions=256, codes=torch.int8)
    gen = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, CFG.vocab, (n,), generator=gen) for n in (4, 40, 17)]
    greedy = serve.generate(prompts, 20)
    assert torch.equal(greedy, serve.generate(prompts, 20, temperature=1.0, top_k=1))

    def drawn(seed):
        g = torch.Generator(device=cuda_device).manual_seed(seed)
        return serve.generate(prompts, 20, g, temperature=1.2, top_k=200, top_p=0.95, min_p=0.01)

    first = drawn(1)
    assert torch.equal(first, drawn(1)) and not torch.equal(first, drawn(2))
    assert bool(((first >= 0) & (first < CFG.vocab)).all())
    assert not serve.seqs and len(serve.pages.free) == 64 and len(serve.open.free) == 64


def test_a_step_captured_in_a_graph_serves_other_lengths(cuda_device):
    """Append, attention and the draw of one step, captured once and replayed
    while the sequences grow through blocks and pages."""
    from dequant_project_b200 import paged_ops
    from dequant_project_b200.sampling import sample_tokens

    dev, n, hq, hkv, d, page = cuda_device, 3, 8, 2, 128, 16
    cos, sin = paged_ops.rope_scaled_tables(d, 1e4, 128, dev)
    gen = torch.Generator(device=dev).manual_seed(1)
    lens0 = [0, 13, 40]

    def state():
        cache = qc.QuantizedCache.empty(24, hkv, page, d, n, device=dev)
        return cache, torch.arange(24, device=dev).int().view(n, 8), torch.arange(n, device=dev).int()

    rows = torch.randn((40, n, (hq + 2 * hkv) * d), generator=gen, device=dev).half()
    draws = torch.rand((40, n), generator=gen, device=dev)
    starts = torch.arange(n + 1, device=dev).int()

    def step(cache, table, slots, qkv, lens, u):
        q = qc.rope_quantized_append(qkv, cos, sin, (lens - 1).long(), cache, table, slots, starts, lens, hq)
        o = qc.quantized_attention(q, cache, table, slots, lens)
        return o, sample_tokens(o.flatten(1), u, top_p=0.9)[0]

    def before(cache, table, slots):
        """What the sequences hold at the beginning."""
        g = torch.Generator(device=dev).manual_seed(2)
        for b, k in enumerate(lens0):
            if k:
                qkv = torch.randn((k, (hq + 2 * hkv) * d), generator=g, device=dev).half()
                qc.rope_quantized_append(qkv, cos, sin, torch.arange(k, device=dev), cache, table[b:b + 1],
                                         slots[b:b + 1], torch.tensor([0, k], device=dev).int(),
                                         torch.tensor([k], device=dev).int(), hq)

    eager = state()
    before(*eager)
    lens = torch.tensor(lens0, device=dev).int()
    want = []
    for i in range(40):
        lens += 1
        want.append(step(*eager, rows[i], lens, draws[i]))
    graphed = state()
    qkv, u, lens = rows[0].clone(), draws[0].clone(), torch.ones(n, device=dev).int()
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*graphed, qkv, lens, u)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        o, t = step(*graphed, qkv, lens, u)
    for x in graphed[0]:
        x.zero_()
    before(*graphed)
    lens.copy_(torch.tensor(lens0, device=dev))
    for i in range(40):
        lens += 1
        qkv.copy_(rows[i])
        u.copy_(draws[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[i][0]) and torch.equal(t, want[i][1])
    assert _native.device_status(dev.index, reset=True) == 0


@pytest.mark.parametrize("codes", [None, torch.int8], ids=str)
def test_a_draw_from_no_numbers_is_not_another_token(cuda_device, codes):
    """-1, drawn from logits that are NaN, gives its sequence NaN and nothing to
    the others, whose steps are those beside an ordinary token, bit for bit."""
    dec = TPDecoder(CFG, QCFG, seed=3, device=cuda_device, batch=4, kv_len=0)
    gen = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, CFG.vocab, (n,), generator=gen) for n in (4, 20, 17)]
    both = []
    for bad in (True, False):
        serve = PagedDecoder(dec, n_pages=64, page_size=16, max_positions=256, codes=codes)
        ids, logits = serve.add(prompts)
        if bad:
            logits[1] = float("nan")
        drawn = serve.sample(logits, torch.Generator(device=cuda_device).manual_seed(2), temperature=0.9, top_p=0.9)
        assert (int(drawn[1]) == -1) == bad
        steps = []
        for _ in range(20):
            logits = serve.step(ids, drawn)
            steps.append(logits[[0, 2]])
            assert bool(logits[1].isnan().all()) == bad and bool(steps[-1].isfinite().all())
            drawn = serve.sample(logits, temperature=0.9, top_k=1)
            assert (int(drawn[1]) == -1) == bad
        both.append(torch.stack(steps))
    assert torch.equal(*both)
    assert _native.device_status(cuda_device.index, reset=True) == 0
