"""Serving path over a paged cache: host logic on the CPU.

A ``PagedDecoder`` (packed prompts, block tables, page allocation, shared
prefix) against ``TPDecoder.step`` run token by token on its contiguous cache:
same weights, same CPU stand-in for the linear layers, so both form the same
fp16 values up to the order of fp32 sums in the attention (2e-3 of the largest
logit, the bound of the decoder's own tests)."""

from __future__ import annotations

import pytest
import torch

from decoder_reference import max_rel_err
from dequant_project_b200 import paged_ops
from dequant_project_b200.decoder import DecoderConfig, TPDecoder
from dequant_project_b200.packer import QuantConfig, dequantize
from dequant_project_b200.paged_decoder import PageAllocator, PagedDecoder

TINY = DecoderConfig(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, intermediate=640, vocab=1000)
QCFG = QuantConfig(4, 64, False)


def cpu_linear(x, pw):
    return (x.float() @ dequantize(pw).float().t()).to(torch.float16)


def make(n_pages=40, page=8, positions=96):
    dec = TPDecoder(TINY, QCFG, seed=3, batch=1, kv_len=0, linear_fn=cpu_linear)
    return PagedDecoder(dec, n_pages, page, positions)


def one_by_one(tokens):
    """Logits after each token, on the contiguous cache."""
    dec = TPDecoder(TINY, QCFG, seed=3, batch=1, kv_len=0, max_new=len(tokens), linear_fn=cpu_linear)
    return torch.cat([dec.step(tokens[i:i + 1], i) for i in range(len(tokens))]).float()


def prompts_of(*lens):
    gen = torch.Generator().manual_seed(sum(lens))
    return [torch.randint(0, TINY.vocab, (n,), generator=gen) for n in lens]


def test_prompts_and_steps_match_the_contiguous_cache():
    serve = make()
    prompts = prompts_of(1, 8, 13, 21)
    ids, logits = serve.add(prompts)
    more = prompts_of(4, 4, 4, 4)
    steps = [serve.step(ids, torch.stack([m[i] for m in more])) for i in range(4)]
    for b, (p, m) in enumerate(zip(prompts, more)):
        ref = one_by_one(torch.cat([p, m]))
        n = len(p)
        assert max_rel_err(logits[b:b + 1].float(), ref[n - 1:n]) < 2e-3
        for i, s in enumerate(steps):
            assert max_rel_err(s[b:b + 1].float(), ref[n + i:n + i + 1]) < 2e-3


def test_sequences_behind_a_prefix():
    serve = make()
    prefix, a, b = prompts_of(16, 3, 9)
    serve.set_prefix(prefix)
    ids, logits = serve.add([a, b])
    tok = torch.tensor([7, 11])
    step = serve.step(ids, tok)
    for i, p in enumerate((a, b)):
        ref = one_by_one(torch.cat([prefix, p, tok[i:i + 1]]))
        assert max_rel_err(logits[i:i + 1].float(), ref[-2:-1]) < 2e-3
        assert max_rel_err(step[i:i + 1].float(), ref[-1:]) < 2e-3


def test_sequences_come_and_go():
    """Pages of a finished sequence serve the next; some sequences step while
    others wait."""
    serve = make(n_pages=6)
    a, b, c = prompts_of(20, 10, 17)
    (ia,), _ = serve.add([a])
    (ib,), _ = serve.add([b])
    with pytest.raises(RuntimeError, match="pages needed"):
        serve.add([c])
    assert len(serve.pages.free) == 1
    serve.free(ia)
    (ic,), logits = serve.add([c])
    assert max_rel_err(logits.float(), one_by_one(c)[-1:]) < 2e-3
    tok = torch.tensor([5])
    assert max_rel_err(serve.step([ib], tok).float(), one_by_one(torch.cat([b, tok]))[-1:]) < 2e-3
    serve.free(ib)
    serve.free(ic)
    assert len(serve.pages.free) == 6


def test_generate_is_greedy_over_steps():
    prompts = prompts_of(5, 2)
    got = make().generate(prompts, 3)
    for b, p in enumerate(prompts):
        seq = p
        for t in range(3):
            nxt = one_by_one(seq)[-1].argmax()
            # Greedy ties aside, the same token wins.
            assert int(got[b, t]) == int(nxt)
            seq = torch.cat([seq, nxt[None]])


def test_rejects_bad_calls():
    serve = make(positions=16)
    with pytest.raises(ValueError, match="1 to 16"):
        serve.add([torch.zeros(0, dtype=torch.int64)])
    with pytest.raises(ValueError, match="1 to 16"):
        serve.add([torch.zeros(17, dtype=torch.int64)])
    with pytest.raises(ValueError, match="whole pages"):
        serve.set_prefix(torch.zeros(5, dtype=torch.int64))
    ids, _ = serve.add([torch.zeros(16, dtype=torch.int64)])
    with pytest.raises(ValueError, match="16 positions"):
        serve.step(ids, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="one token for each"):
        serve.step(ids + ids, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="before any sequence"):
        serve.set_prefix(torch.zeros(8, dtype=torch.int64))


def test_page_allocator():
    a = PageAllocator(4)
    assert a.take(3) == [0, 1, 2]
    with pytest.raises(RuntimeError, match="2 pages needed, 1 free"):
        a.take(2)
    a.give([1])
    assert sorted(a.take(2)) == [1, 3] and a.take(0) == []


@pytest.mark.parametrize("scaling,check", [
    (None, lambda f, b: torch.equal(f, b)),
    ({"type": "linear", "factor": 4.0}, lambda f, b: torch.allclose(f, b / 4)),
    ({"type": "dynamic", "factor": 2.0, "original": 64}, lambda f, b: bool((f[1:] < b[1:]).all() and f[0] == b[0])),
    ({"type": "banded", "factor": 8.0, "original": 64, "low": 1.0, "high": 4.0},
     lambda f, b: bool(f[0] == b[0] and torch.isclose(f[-1], b[-1] / 8) and (f <= b).all())),
])
def test_rope_scaling(scaling, check):
    """The frequencies behind the tables: at position 1 the angle is the
    frequency itself (all below pi here)."""
    cos, sin = paged_ops.rope_scaled_tables(64, 10000.0, 128, "cpu", scaling=scaling)
    assert cos.shape == sin.shape == (128, 32) and cos.dtype == torch.float32
    freq = torch.atan2(sin[1].double(), cos[1].double())
    base = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    base = torch.atan2(base.sin().float().double(), base.cos().float().double())
    assert check(freq, base)


def test_rope_tables_reject_bad_arguments():
    for kw in ({"rotary_dim": 3}, {"rotary_dim": 66}, {"scaling": {"type": "other"}},
               {"scaling": {"type": "linear", "factor": 0.5}}):
        with pytest.raises(ValueError):
            paged_ops.rope_scaled_tables(64, 1e4, 8, "cpu", **kw)


def _serve(world):
    import socket

    import torch.multiprocessing as mp

    import paged_workers
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    procs = [ctx.Process(target=paged_workers.serve, args=(r, world, port, queue)) for r in range(world)]
    for p in procs:
        p.start()
    got = {}
    for _ in procs:
        rank, logits, err = queue.get(timeout=120)
        assert err is None, err
        got[rank] = torch.from_numpy(logits)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    return got


def test_two_ranks_serve_what_one_does():
    """Heads, intermediate and vocabulary split over two gloo ranks: every rank
    gathers the logits of the single-rank run (sums of two partials instead of
    one: the decoder tests' bound)."""
    one, two = _serve(1)[0], _serve(2)
    assert torch.equal(two[0], two[1])
    assert max_rel_err(two[0], one) < 5e-3
