"""Serving with a cache held in 8 bits and with drawn tokens: host logic on the
CPU.

The first layer's keys and values depend on the tokens alone, so a quantised
decoder's first cache has to hold, bit for bit, the codes of what the 16-bit
decoder's first cache holds. Its logits are those of a model whose cached values
are off by half a step (2^-8 of a block's largest for int8, 2^-4 of a value for
e4m3), which two layers of random weights turn into a few per cent of the
largest logit: a bound that only a wrong cache, table or length breaks."""

from __future__ import annotations

import pytest
import torch

from decoder_reference import max_rel_err
from dequant_project_b200 import quantized_cache as qc
from dequant_project_b200.decoder import DecoderConfig, TPDecoder
from dequant_project_b200.paged_decoder import PagedDecoder
from test_paged_decoder import QCFG, cpu_linear
from test_paged_decoder_errors import Failing

# Heads of 64, which an 8-bit cache's blocks of 16 positions go with.
CFG = DecoderConfig(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, intermediate=640, vocab=1000)
BOUND = {torch.int8: 0.05, torch.float8_e4m3fn: 0.25}


def make(codes=None, n_pages=40, page=16, linear=cpu_linear, **kw):
    dec = TPDecoder(CFG, QCFG, seed=3, batch=1, kv_len=0, linear_fn=linear)
    return PagedDecoder(dec, n_pages, page, 192, codes=codes, **kw)


def prompts_of(*lens):
    gen = torch.Generator().manual_seed(sum(lens))
    return [torch.randint(0, CFG.vocab, (n,), generator=gen) for n in lens]


def cached(serve, i, layer=0):
    """16-bit rows [kv heads, len, D] of a sequence's keys and values."""
    s = serve.seqs[i]
    pages, n = serve.prefix_pages + s["pages"], serve.prefix_len + s["len"]
    t = torch.arange(n)
    at = torch.tensor(pages)[t // serve.page]
    if serve.codes is None:
        return [p[layer][at, :, t % serve.page].transpose(0, 1) for p in (serve.k, serve.v)]
    table = torch.tensor([pages], dtype=torch.int32)
    return [qc._rows(serve.cache[layer], w, table[0], s["open"], n) for w in (0, 1)]


@pytest.mark.parametrize("codes", list(BOUND), ids=str)
@pytest.mark.parametrize("block,prefix", [(16, 0), (32, 0), (16, 48)])
def test_against_the_16_bit_cache(codes, block, prefix):
    page = 32 if block == 32 else 16
    plain, serve = make(page=page), make(codes, page=page, block=block)
    toks, more = prompts_of(1, 16, 33, 70), prompts_of(20, 20, 20, 20)
    results = []
    for s in (plain, serve):
        if prefix:
            s.set_prefix(prompts_of(prefix)[0])
        ids, logits = s.add(toks)
        results.append([logits] + [s.step(ids, torch.stack([m[i] for m in more])) for i in range(20)])
    for a, b in zip(*results):
        assert max_rel_err(b.float(), a.float()) < BOUND[codes]
    for i in ids:
        for want, got in zip(cached(plain, i), cached(serve, i)):
            n = want.shape[1] - want.shape[1] % block
            c, scale = qc.quantize_block(want[:, :n].unflatten(1, (-1, block)), codes)
            assert torch.equal(got[:, :n], (c.float() * scale[..., None, None]).flatten(1, 2))
            assert torch.equal(got[:, n:], want[:, n:].float())


def test_open_blocks_are_given_back():
    serve = make(torch.int8, max_seqs=3)
    ids, _ = serve.add(prompts_of(5, 40, 16))
    assert sorted(serve.seqs[i]["open"] for i in ids) == [0, 1, 2]
    with pytest.raises(RuntimeError, match="1 open blocks needed, 0 free"):
        serve.add(prompts_of(3))
    free = len(serve.pages.free)
    serve.free(ids[1])
    assert len(serve.pages.free) == free + 3
    (again,), _ = serve.add(prompts_of(3))
    assert serve.seqs[again]["open"] == 1
    for i in (ids[0], ids[2], again):
        serve.free(i)
    assert sorted(serve.open.free) == [0, 1, 2] and len(serve.pages.free) == 40


@pytest.mark.parametrize("after", [1, 4, 7])
def test_a_pass_that_raises_leaves_all_as_it_was(after):
    linear = Failing()
    serve, other = make(torch.int8, linear=linear), make(torch.int8)
    toks = prompts_of(15, 20)
    linear.arm(after)
    with pytest.raises(RuntimeError, match="no memory"):
        serve.add(toks)
    assert len(serve.pages.free) == 40 and len(serve.open.free) == 64 and not serve.seqs
    ids, _ = serve.add(toks)
    other.add(toks)
    for step in range(3):  # the first one completes a block
        tok = torch.tensor([5 + step, 9])
        linear.arm(after)
        with pytest.raises(RuntimeError, match="no memory"):
            serve.step(ids, torch.tensor([7, 8]))
        assert torch.equal(serve.step(ids, tok), other.step(ids, tok))


def test_generate_draws_what_its_generator_says():
    serve = make(torch.int8)
    prompts = prompts_of(4, 9, 17)
    greedy = serve.generate(prompts, 6)
    assert torch.equal(greedy, serve.generate(prompts, 6, temperature=0.0))
    assert torch.equal(greedy, serve.generate(prompts, 6, temperature=1.0, top_k=1))
    draws = [serve.generate(prompts, 6, torch.Generator().manual_seed(s), temperature=1.5, top_p=0.95) for s in (1, 1, 2)]
    assert torch.equal(draws[0], draws[1]) and not torch.equal(draws[0], draws[2])
    assert not serve.seqs and len(serve.pages.free) == 40
    serve.dec.world = 2
    with pytest.raises(ValueError, match="seeded alike"):
        serve.sample(torch.zeros((1, 5)), temperature=1.0)


def _serve(world):
    import socket

    import torch.multiprocessing as mp

    import paged_workers
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    procs = [ctx.Process(target=paged_workers.serve_quantized, args=(r, world, port, queue)) for r in range(world)]
    for p in procs:
        p.start()
    got = {}
    for _ in procs:
        rank, results, err = queue.get(timeout=120)
        assert err is None, err
        got[rank] = [torch.from_numpy(x) for x in results]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    return got


def test_two_ranks_serve_what_one_does():
    """Heads over two gloo ranks, each with open blocks of its own: both gather
    the same logits and draw the same tokens. One rank's logits differ by the order
    of sums, which can turn a code over: as much as rounding to codes does at most."""
    one, two = _serve(1)[0], _serve(2)
    assert torch.equal(two[0][0], two[1][0]) and torch.equal(two[0][1], two[1][1])
    assert max_rel_err(two[0][0], one[0]) < BOUND[torch.int8]
    for _, draws in (one, two[0]):
        assert draws.shape == (2, 8) and bool(((draws >= 0) & (draws < 1001)).all())
