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
