"""Bounded waits of the paged decode kernel end in an error status, not a hang,
and the kernel that joins its pieces finds every item described.

``dqg_debug_paged_starved`` runs the kernels with warps that do nothing: the
copying warp (every wait for data runs out), or one consumer warp (the others
go on until the ring is not emptied any more, and meet it at their barriers all
the same). The calls must return, write NaN for what was given up and nothing
outside the outputs, on scratch memory of any contents, and leave the context
usable."""

from __future__ import annotations

import pytest
import torch

from dequant_project_b200 import _native, paged_ops
from test_paged_ops_gpu import make_cache

pytestmark = pytest.mark.gpu

WAIT_NS = 2_000_000
COPIES = 16


def starved_call(q, k, v, pre, prefix, table, lens, ws, out, mask):
    kv = _native.PagedKV(k.data_ptr(), v.data_ptr(), *k.shape, *k.stride()[:3], 0)
    _native.check(_native.lib().dqg_debug_paged_starved(
        q.data_ptr(), q.stride(0), q.stride(1), q.shape[0], q.shape[1], kv, pre.data_ptr(), pre.shape[0], prefix,
        table.data_ptr(), table.shape[1], table.stride(0), lens.data_ptr(), 0.1, out.data_ptr(), ws.data_ptr(),
        ws.numel(), mask, WAIT_NS, torch.cuda.current_stream().cuda_stream))


CASES = [
    # prefix, lengths, hq, hkv
    (0, [700, 0, 33], 8, 2),               # items cut over many CTAs
    (0, [40] * 300, 8, 2),                 # many whole items a CTA
    (0, [500, 70], 40, 1),                 # several row blocks
    (300, [90, 0, 5], 8, 2),               # a prefix that the decode kernel streams
    (300, list(range(60)), 64, 8),         # a prefix that the prompt kernel takes
]


@pytest.mark.parametrize("mask", [COPIES, 1, 4, 10], ids=["copies", "warp 0", "warp 2", "two warps"])
@pytest.mark.parametrize("prefix,lens,hq,hkv", CASES, ids=lambda x: str(x)[:24])
def test_starved_kernels_give_up_and_report(cuda_device, prefix, lens, hq, hkv, mask):
    gen = torch.Generator(device=cuda_device).manual_seed(prefix + len(lens))
    d, page = 128, 16
    k, v, table = make_cache(gen, lens + [max(prefix, 1)], hkv, d, page, torch.float16, cuda_device)
    pre, tab = table[-1].contiguous(), table[:-1].contiguous()
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    q = torch.randn((len(lens), hq, d), generator=gen, device=cuda_device).half()
    size = q.numel()
    guarded = torch.full((3 * size,), 7.0, dtype=torch.float16, device=cuda_device)
    out = guarded[size:2 * size]
    ws = paged_ops.shared_prefix_workspace(len(lens), hq, hkv, d, prefix, cuda_device).fill_(255)
    torch.cuda.synchronize()
    _native.device_status(cuda_device.index, reset=True)
    starved_call(q, k, v, pre, prefix, tab, n, ws, out, mask)
    torch.cuda.synchronize()  # returns: every wait gave up after WAIT_NS
    status = _native.device_status(cuda_device.index, reset=True)
    assert torch.isnan(out.float()).all()
    assert (guarded[:size] == 7.0).all() and (guarded[2 * size:] == 7.0).all()
    if mask == COPIES:
        assert status & 1, f"status {status:#x}: no wait reported giving up"
    # The context is still usable and the next call, on the same scratch, is right.
    want = paged_ops.shared_prefix_attention(q, k, v, pre, prefix, tab, n)
    assert torch.isfinite(want).all()
    assert torch.equal(paged_ops.shared_prefix_attention(q, k, v, pre, prefix, tab, n, workspace=ws), want)
    assert _native.device_status(cuda_device.index) == 0


def test_rejects_bad_arguments(cuda_device):
    z = torch.zeros(64, dtype=torch.float16, device=cuda_device)
    t = torch.zeros((1, 1), dtype=torch.int32, device=cuda_device)
    k = torch.zeros((1, 1, 16, 64), dtype=torch.float16, device=cuda_device)
    for mask in (0, 32):
        with pytest.raises(RuntimeError, match="starved must be"):
            starved_call(z.view(1, 1, 64), k, k, t[0], 0, t, t[0], z, z, mask)
