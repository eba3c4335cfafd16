"""A serving pass that raises (out of memory, a rejected argument, a collective
that fails) leaves a ``PagedDecoder`` as it was: no page is lost, no sequence is
longer than what its layers have stored, and the same call can be made again."""

from __future__ import annotations

import pytest
import torch

from decoder_reference import max_rel_err
from dequant_project_b200.decoder import TPDecoder
from dequant_project_b200.paged_decoder import PagedDecoder
from test_paged_decoder import QCFG, TINY, cpu_linear, one_by_one, prompts_of


class Failing:
    """The CPU stand-in for the linear layers, raising at call number ``at``."""

    def __init__(self):
        self.calls, self.at = 0, -1

    def __call__(self, x, pw):
        self.calls += 1
        if self.calls == self.at:
            raise RuntimeError("no memory")
        return cpu_linear(x, pw)

    def arm(self, after):
        self.at = self.calls + after


def make(n_pages=12, page=8, positions=96):
    linear = Failing()
    dec = TPDecoder(TINY, QCFG, seed=3, batch=1, kv_len=0, linear_fn=linear)
    return PagedDecoder(dec, n_pages, page, positions), linear


@pytest.mark.parametrize("after", [1, 4, 7])
def test_step(after):
    serve, linear = make()
    a, b = prompts_of(8, 13)  # the first one's next token takes a new page
    ids, _ = serve.add([a, b])
    free = sorted(serve.pages.free)
    tok = torch.tensor([5, 9])
    linear.arm(after)
    with pytest.raises(RuntimeError, match="no memory"):
        serve.step(ids, tok)
    assert sorted(serve.pages.free) == free
    assert [serve.seqs[i]["len"] for i in ids] == [8, 13]
    assert [len(serve.seqs[i]["pages"]) for i in ids] == [1, 2]
    got = serve.step(ids, tok).float()
    for i, p in enumerate((a, b)):
        assert max_rel_err(got[i:i + 1], one_by_one(torch.cat([p, tok[i:i + 1]]))[-1:]) < 2e-3


@pytest.mark.parametrize("after", [1, 5])
def test_add_and_set_prefix(after):
    serve, linear = make()
    linear.arm(after)
    prefix, a, b = prompts_of(16, 3, 9)
    with pytest.raises(RuntimeError, match="no memory"):
        serve.set_prefix(prefix)
    assert len(serve.pages.free) == 12 and serve.prefix_len == 0 and not serve.prefix_pages
    serve.set_prefix(prefix)
    assert len(serve.pages.free) == 10
    linear.arm(after)
    with pytest.raises(RuntimeError, match="no memory"):
        serve.add([a, b])
    assert len(serve.pages.free) == 10 and not serve.seqs
    ids, logits = serve.add([a, b])
    for i, p in enumerate((a, b)):
        assert max_rel_err(logits[i:i + 1].float(), one_by_one(torch.cat([prefix, p]))[-1:]) < 2e-3


def test_generate():
    serve, linear = make(n_pages=3)
    with pytest.raises(RuntimeError, match="pages needed"):  # no page for the third step
        serve.generate(prompts_of(14, 6), 5)
    assert len(serve.pages.free) == 3 and not serve.seqs
    assert serve.generate(prompts_of(3, 2), 0).shape == (2, 0)
    assert len(serve.pages.free) == 3 and not serve.seqs


@pytest.mark.parametrize("bad", [-1, TINY.vocab])
def test_tokens_outside_the_vocabulary(bad):
    serve, _ = make()
    tok = torch.tensor([3, bad, 5, 6, 7, 8, 9, 10])
    for call in (lambda: serve.set_prefix(tok), lambda: serve.add([tok[:1], tok])):
        with pytest.raises(ValueError, match=f"tokens must be in .*, got {bad}"):
            call()
    ids, _ = serve.add([tok[:1]])
    with pytest.raises(ValueError, match=f"got {bad}"):
        serve.step(ids, tok[1:2])
    assert serve.seqs[ids[0]]["len"] == 1 and len(serve.pages.free) == 11
