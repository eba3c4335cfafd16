"""Values that a causal mask hides, in the torch formulas that CPU tensors take:
rows that do not see a non-finite value give what they give with a zero there,
rows that see it take it."""

from __future__ import annotations

import pytest
import torch

from dequant_project_b200 import paged_ops


@pytest.mark.parametrize("ql,kl", [(5, 20), (20, 20), (9, 4)])
@pytest.mark.parametrize("x", [float("nan"), float("inf"), float("-inf")])
def test_hidden_values_do_not_matter(x, ql, kl):
    gen = torch.Generator().manual_seed(ql + kl)
    hkv, page, d = 2, 16, 64
    k, v = (torch.randn((3, hkv, page, d), generator=gen).half() for _ in range(2))
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    lens, starts = torch.tensor([kl], dtype=torch.int32), torch.tensor([0, ql], dtype=torch.int32)
    q = torch.randn((ql, 4, d), generator=gen).half()
    bad, clean = v.clone(), v.clone()
    t = kl - 2
    bad[table[0, t // page].long(), :, t % page, 7] = x
    clean[table[0, t // page].long(), :, t % page, 7] = 0.0
    want = paged_ops.prompt_attention(q, k, clean, table, starts, lens)
    got = paged_ops.prompt_attention(q, k, bad, table, starts, lens)
    sees = torch.arange(ql) + kl - ql >= t
    assert torch.equal(got[~sees], want[~sees])
    assert torch.equal(got[sees][..., :7], want[sees][..., :7])
    hit = got[sees][..., 7].float()
    assert bool((torch.isnan(hit) if x != x else hit == x).all())
    assert torch.isfinite(want.float()).all()
