"""Prompt rows of a sequence without positions are zeros, whatever a product
before them has left in the tensor cores' memory."""

from __future__ import annotations

import pytest
import torch

from dequant_project_b200 import paged_ops
from dequant_project_b200 import quantized_cache as qc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("eight_bits", [False, True], ids=["16 bits", "8 bits"])
def test_rows_without_keys_behind_values_that_are_not_numbers(cuda_device, eight_bits, d, causal):
    hq, hkv, page, n = 16, 8, 16, 4096

    def ints(*values):
        return torch.tensor(values, dtype=torch.int32, device=cuda_device)

    pages = n // page
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    q = torch.randn((n, hq, d), device=cuda_device).half()
    k = torch.randn((pages, hkv, page, d), device=cuda_device).half()
    v = torch.full_like(k, float("nan"))
    cache = qc.QuantizedCache.empty(pages, hkv, page, d, 1, device=cuda_device)
    cache.v_scale.fill_(float("nan"))

    def attend(q, starts, lens):
        if eight_bits:
            return qc.quantized_prompt_attention(q, cache, table, ints(0), starts, lens, pages, causal=causal)
        return paged_ops.prompt_attention(q, k, v, table, starts, lens, causal=causal)

    for rows in (1, 5, 300):
        assert bool(attend(q, ints(0, n), ints(n)).isnan().all())  # on every SM
        out = attend(q[:rows], ints(0, rows), ints(0))
        assert bool((out == 0).all())


@pytest.mark.parametrize("fill", [0, 0x3c, 0x7e, 255])
@pytest.mark.parametrize("hq,hkv,d", [(32, 2, 64), (16, 8, 128), (1, 1, 64)])
def test_rows_without_keys_on_scratch_of_any_contents(cuda_device, hq, hkv, d, fill):
    cache = qc.QuantizedCache.empty(4, hkv, 64, d, 3, block=32, device=cuda_device)
    gen = torch.Generator(device=cuda_device).manual_seed(hq)
    for x in cache[4:]:
        x.copy_(torch.randn(x.shape, generator=gen, device=cuda_device))
    q = torch.randn((8, hq, d), generator=gen, device=cuda_device).half()

    def ints(*values):
        return torch.tensor(values, dtype=torch.int32, device=cuda_device)

    table = ints(0, 1, 2)[:, None]
    for starts, lens, pages in (((0, 3, 3, 8), (0, 0, 0), 0), ((0, 3, 4, 8), (0, 1, 0), 1), ((0, 1, 4, 8), (5, 0, 7), 2)):
        ws = qc.quantized_prompt_workspace(cache, 3, 1, pages).fill_(fill)
        out = qc.quantized_prompt_attention(q, cache, table, ints(0, 1, 2), ints(*starts), ints(*lens), pages,
                                            workspace=ws)
        assert bool(out.isfinite().all())
        for b, n in enumerate(lens):
            if n == 0:
                assert bool((out[starts[b]:starts[b + 1]] == 0).all())
