"""Decode attention behind prefixes on both sides of the rule that says which
kernel reads the prefix: a short one is streamed with the sequences' own pages for
up to two 16-row tiles, a long one for one tile only. Bounds as in
test_paged_ops_gpu."""

from __future__ import annotations

import math

import pytest
import torch

from dequant_project_b200 import _native, paged_ops
from test_paged_ops_gpu import attend64, check_attention, make_cache, rows64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefix,n,hq,hkv,d", [
    (6144, 17, 32, 32, 128),    # 96 MiB: two tiles, streamed
    (6145, 17, 32, 32, 128),    # more: by the prompt kernel
    (12000, 32, 32, 32, 128),
    (12000, 16, 32, 32, 128),   # one tile: streamed
    (12000, 3, 8, 1, 64),
])
def test_prefix(cuda_device, prefix, n, hq, hkv, d):
    gen = torch.Generator(device=cuda_device).manual_seed(prefix + n)
    lens = [(37 * i) % 130 for i in range(n)]
    k, v, table = make_cache(gen, lens + [prefix], hkv, d, 64, torch.float16, cuda_device, fill=float("nan"))
    own, shared = table[:-1].contiguous(), table[-1].contiguous()
    q = torch.randn((n, hq, d), generator=gen, device=cuda_device).half()
    kv_lens = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    ws = paged_ops.shared_prefix_workspace(n, hq, hkv, d, prefix, cuda_device).fill_(255)
    out = paged_ops.shared_prefix_attention(q, k, v, shared, prefix, own, kv_lens, workspace=ws)
    for i in range(0, n, 5):
        kk, vv = (torch.cat([rows64(p, shared, prefix), rows64(p, own[i], lens[i])]) for p in (k, v))
        ref = attend64(q[i:i + 1], kk, vv, kv_lens[i:i + 1] + prefix, 1 / math.sqrt(d))
        check_attention(out[i:i + 1], ref, float(vv.abs().max()), torch.float16)
    assert torch.equal(paged_ops.shared_prefix_attention(q, k, v, shared, prefix, own, kv_lens), out)
    assert _native.device_status(cuda_device.index) == 0
