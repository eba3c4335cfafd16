"""Calls of the paged operators with one input at a time that requires a
gradient, for the tests on either device. Not a test module."""

from __future__ import annotations

import torch

from dequant_project_b200 import paged_ops


def calls(device):
    """(name, call, its floating-point inputs by name)"""
    gen = torch.Generator().manual_seed(0)

    def r(*shape, dtype=torch.float16):
        return torch.randn(shape, generator=gen).to(dtype).to(device)

    def i(*values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device=device)

    pools = {"k_pages": r(3, 2, 16, 64), "v_pages": r(3, 2, 16, 64)}
    table, lens, i64 = i([1, 2], [0, 2]), i(20, 3), torch.int64
    return [
        ("append", lambda **t: paged_ops.rope_paged_append(positions=i(0, 1, dtype=i64), slots=i(17, 3, dtype=i64),
                                                           n_q_heads=4, **t),
         {"qkv": r(2, 8 * 64), "cos": r(8, 32, dtype=torch.float32), "sin": r(8, 32, dtype=torch.float32),
          "q_norm": r(64), "k_norm": r(64), **pools}),
        ("decode", lambda **t: paged_ops.paged_attention(block_table=table, kv_lens=lens, **t),
         {"q": r(2, 4, 64), **pools}),
        ("prompt", lambda **t: paged_ops.prompt_attention(block_table=table, q_starts=i(0, 1, 2), kv_lens=lens, **t),
         {"q": r(2, 4, 64), **pools}),
        ("shared", lambda **t: paged_ops.shared_prefix_attention(prefix_table=i(2), prefix_len=9, block_table=table,
                                                                 kv_lens=lens, **t),
         {"q": r(2, 4, 64), **pools}),
    ]


def check(device):
    for name, call, inputs in calls(device):
        out = call(**inputs)
        assert not out.requires_grad
        for one in inputs:
            changed = {k: t.clone().requires_grad_(k == one) for k, t in inputs.items()}
            try:
                call(**changed)
            except RuntimeError as exc:
                assert "forward only" in str(exc), (name, one, exc)
            else:
                raise AssertionError(f"{name}: {one} required a gradient that was dropped")
            with torch.no_grad():
                assert torch.equal(call(**changed), out), (name, one)
    # The pages' versions rise with each append, by which autograd knows.
    _, append, inputs = calls(device)[0]
    before = [inputs[n]._version for n in ("k_pages", "v_pages")]
    append(**inputs)
    assert all(inputs[n]._version > b for n, b in zip(("k_pages", "v_pages"), before))
    with torch.inference_mode():
        append(**{n: t.clone() for n, t in inputs.items()})
