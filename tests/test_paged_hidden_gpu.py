"""Values that a causal mask hides, on the GPU: whatever they hold, rows that
do not see them give what they give with zeros there, bit for bit, and a row
that sees a non-finite value takes it as the sum over its keys does. (The
products run over whole blocks of keys for whole tiles of rows, where a zero
weight times an infinity would not be zero.)"""

from __future__ import annotations

import pytest
import torch

from dequant_project_b200 import _native, paged_ops
from test_paged_ops_gpu import TYPES, make_cache

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")

CASES = [
    # query lengths, key lengths, hq, hkv, d, page
    ([128], [200], 1, 1, 128, 16),            # a row's last key one block before the hidden one
    ([300], [700], 2, 2, 128, 64),            # two tiles that see different parts of the last blocks
    ([300], [700], 16, 2, 64, 16),
    ([200], [150], 4, 2, 128, 16),            # rows that see no key at all
    ([1000], [40], 2, 1, 64, 32),             # whole tiles that see none
    ([40], [5000], 8, 1, 128, 32),            # one item, cut into pieces
    ([1, 130, 0, 77], [9, 130, 5, 300], 28, 4, 128, 128),
    ([200, 333], [260, 333], 3, 1, 64, 256),
]


def place(v, table, b, t, page, col, x):
    v[table[b, t // page].long(), :, t % page, col] = x


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("ql,kl,hq,hkv,d,page", CASES, ids=lambda v: str(v)[:40])
def test_prompt(cuda_device, ql, kl, hq, hkv, d, page, causal, dtype):
    gen = torch.Generator(device=cuda_device).manual_seed(sum(ql) + hq)
    k, v, table = make_cache(gen, kl, hkv, d, page, dtype, cuda_device, fill=NAN)
    starts = torch.tensor([0] + ql, device=cuda_device).cumsum(0).int()
    lens = torch.tensor(kl, dtype=torch.int32, device=cuda_device)
    q = torch.randn((sum(ql), hq, d), generator=gen, device=cuda_device).to(dtype)
    bad, clean = v.clone(), v.clone()
    taint = torch.zeros((sum(ql), d), dtype=torch.float64, device=cuda_device)
    for b, (m, n) in enumerate(zip(ql, kl)):
        # The last blocks' positions: hidden from some rows, seen by others.
        at = sorted({max(0, n - 1 - back) for back in (0, 1, m // 4, m // 2, m - 1, m, 49, 50)})
        for i, t in enumerate(at):
            x, col = ((INF, 5), (NAN, 17), (-INF, 33), (INF, 33))[i % 4]
            place(bad, table, b, t, page, col, x)
            place(clean, table, b, t, page, col, 0.0)
            for r in range(m):
                if not causal or t < n - m + r + 1:
                    taint[int(starts[b]) + r, col] += x
    want = paged_ops.prompt_attention(q, k, clean, table, starts, lens, causal=causal)
    assert torch.isfinite(want.float()).all()
    got = paged_ops.prompt_attention(q, k, bad, table, starts, lens, causal=causal)
    taint = taint[:, None].expand(-1, hq, -1)
    hit = ~torch.isfinite(taint)
    assert torch.equal(got[~hit], want[~hit])
    assert torch.equal(got[hit].double().nan_to_num(7.0, 1.0, -1.0), taint[hit].nan_to_num(7.0, 1.0, -1.0))
    for _ in range(2):
        again = paged_ops.prompt_attention(q, k, bad, table, starts, lens, causal=causal)
        assert torch.equal(again.view(torch.int16), got.view(torch.int16))
    assert _native.device_status(cuda_device.index) == 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", [40, 300])
def test_prefix_of_many_rows(cuda_device, rows, dtype):
    """A non-finite value in a prefix's last, partial block reaches every
    sequence; what lies behind the prefix none."""
    gen = torch.Generator(device=cuda_device).manual_seed(rows)
    prefix, own, hq, hkv, d, page = 333, 20, 8, 1, 128, 16
    k, v, table = make_cache(gen, [own] * rows + [prefix], hkv, d, page, dtype, cuda_device, fill=NAN)
    lens = torch.full((rows,), own, dtype=torch.int32, device=cuda_device)
    q = torch.randn((rows, hq, d), generator=gen, device=cuda_device).to(dtype)
    pre, tab = table[-1].contiguous(), table[:-1].contiguous()
    bad, clean = v.clone(), v.clone()
    for t, col, x in ((332, 3, INF), (300, 70, NAN), (100, 9, -INF)):
        place(bad, table, rows, t, page, col, x)
        place(clean, table, rows, t, page, col, 0.0)
    want = paged_ops.shared_prefix_attention(q, k, clean, pre, prefix, tab, lens)
    got = paged_ops.shared_prefix_attention(q, k, bad, pre, prefix, tab, lens)
    assert torch.isposinf(got[..., 3]).all() and torch.isnan(got[..., 70]).all() and torch.isneginf(got[..., 9]).all()
    keep = [c for c in range(d) if c not in (3, 70, 9)]
    assert torch.isfinite(want.float()).all() and torch.equal(got[..., keep], want[..., keep])
