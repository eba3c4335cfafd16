"""Row starts of packed prompts that are out of order or range, on the GPU: the
sequences that they bound have no rows, which is reported; the others, whose
starts are in order, are served."""

from __future__ import annotations

import pytest
import torch

from dequant_project_b200 import _native, paged_ops
from test_paged_ops_gpu import make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("many", [False, True], ids=["one scan", "scans"])
@pytest.mark.parametrize("starts,served", [
    ([0, 5, 2, 7], (0, 2)),        # out of order
    ([0, 3, 3, 8], (0, 1)),        # past the last row
    ([-4, 2, 4, 7], (1, 2)),       # before the first
    ([0, 1 << 30, 4, 7], (2,)),
])
def test_starts_out_of_order_are_reported(cuda_device, starts, served, many):
    gen = torch.Generator(device=cuda_device).manual_seed(len(served))
    t, lens = 7, [40, 33, 64]
    if many:  # more sequences than one scan takes
        starts, lens = starts + [t] * 40, lens + [9] * 40
    k, v, table = make_cache(gen, lens, 2, 64, 16, torch.float16, cuda_device)
    q = torch.randn((t, 4, 64), generator=gen, device=cuda_device).half()
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    _native.device_status(cuda_device.index, reset=True)
    out = paged_ops.prompt_attention(q, k, v, table, torch.tensor(starts, dtype=torch.int32, device=cuda_device), n)
    torch.cuda.synchronize()
    assert _native.device_status(cuda_device.index, reset=True) == 2
    for b in served:
        lo, hi = starts[b], starts[b + 1]
        if any(starts[c] < hi and starts[c + 1] > lo for c in served if c != b):
            continue  # rows that two sequences claim belong to neither
        own = torch.tensor([0, hi - lo], dtype=torch.int32, device=cuda_device)
        want = paged_ops.prompt_attention(q[lo:hi], k, v, table[b:b + 1], own, n[b:b + 1])
        assert torch.equal(out[lo:hi], want)
    assert _native.device_status(cuda_device.index) == 0
