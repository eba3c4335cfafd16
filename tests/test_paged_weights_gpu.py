"""The range of the softmax weights that the paged operators hold in 16 bits for
the product with the values, on the GPU.

Outputs are rounded once (u), and so is each weight; the largest weight of a row
is 2^7 at least (prompt kernel) or 2^15 (decode), so that below fp16's smallest
normal number (2^-14, absolute error 2^-25) a weight loses at most 2^-32, or
2^-40, of the largest one. Exponentials and fp32 sums add below 2^-14 of max|v|.
"""

from __future__ import annotations

import math

import pytest
import torch

from dequant_project_b200 import paged_ops
from test_paged_ops_gpu import TYPES, U

pytestmark = pytest.mark.gpu


def check(out, ref, v_max, u, slack):
    err = (out.double() - ref).abs()
    lim = u * ref.abs() + slack * v_max + 1e-7
    assert bool((err <= lim).all()), f"max excess {float((err - lim).max()):.3e}, max error {float(err.max()):.3e}"


# One dominating key and a long flat tail, whose weights a 16-bit type with a
# small exponent range would round away: each is 2^-25.5 of the largest one, and
# at 131072 keys they hold 0.27 % of the sum. Enough rows that nothing is cut
# into pieces with maxima of their own.
TAIL, LOG2 = 131072, 25.5


def sink(device, dtype, where, d=64, page=256):
    """Keys of one head; the sink's value is 0, the tail's are 1."""
    order = torch.randperm(TAIL // page, generator=torch.Generator().manual_seed(where)).int().to(device)
    k = torch.zeros((TAIL // page, 1, page, d), dtype=dtype, device=device)
    v = torch.ones_like(k)
    at = order[where // page].long()
    k[at, :, where % page, 0] = 8.0
    v[at, :, where % page] = 0.0
    return k, v, order


def sink_query(device, dtype, rows, heads, d=64):
    q = torch.zeros((rows, heads, d), dtype=dtype, device=device)
    q[..., 0] = LOG2 * math.log(2.0) / 8.0
    return q


def tail_share(q, n):
    """The output: the tail's part of the sum, in 64 bits (scale 1)."""
    w = (n - 1) * math.exp(-8.0 * float(q[0, 0, 0]))
    return w / (1.0 + w)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("where", [0, 70000, TAIL - 1])
@pytest.mark.parametrize("call", ["decode", "prompt", "prefix"])
def test_a_flat_tail_behind_one_large_weight(cuda_device, call, where, dtype):
    """What a weight loses below the smallest one that 16 bits hold adds up over
    the keys: at most 2^-32 of the largest weight for each (prompt kernel; decode
    2^-40), 2^-15 of max|v| for this many."""
    k, v, order = sink(cuda_device, dtype, where)
    pages = order.shape[0]
    if call == "decode":
        rows = 600
        q = sink_query(cuda_device, dtype, rows, 1)
        lens = torch.full((rows,), TAIL, dtype=torch.int32, device=cuda_device)
        out = paged_ops.paged_attention(q, k, v, order.expand(rows, pages).contiguous(), lens, scale=1.0)
    elif call == "prompt":
        rows = 148 * 256
        q = sink_query(cuda_device, dtype, rows, 1)
        starts = torch.tensor([0, rows], dtype=torch.int32, device=cuda_device)
        lens = torch.tensor([TAIL], dtype=torch.int32, device=cuda_device)
        out = paged_ops.prompt_attention(q, k, v, order[None], starts, lens, causal=False, scale=1.0)
    else:
        rows = 148 * 64
        q = sink_query(cuda_device, dtype, rows, 4)
        lens = torch.zeros(rows, dtype=torch.int32, device=cuda_device)
        out = paged_ops.shared_prefix_attention(q, k, v, order, TAIL, order[:1].expand(rows, 1).contiguous(),
                                                lens, scale=1.0)
    ref = torch.full(out.shape, tail_share(q, TAIL), dtype=torch.float64, device=cuda_device)
    check(out, ref, 1.0, 2 * U[dtype], 2.0 ** -13)
