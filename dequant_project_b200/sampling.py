"""The draw of the next token from rows of logits.

CUDA tensors go through the sm_100a kernel of libdequant_b200.so on torch's
current stream (``binding/paged_binding.cpp``); if it is missing the call
raises. CPU tensors take the same formulas in torch, in 64 bits: that branch
exists for the host-logic tests and is never taken for a CUDA tensor.

The reference has no counterpart: its path ends at the LM head's GEMV
(KrishnaI2424/Dequant_Project ``dequant/quant_linear.py:150-162``).
"""

from __future__ import annotations

import torch

from dequant_project_b200 import paged_ops as paged


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: torch.Tensor | float = 1.0,
                  top_k: torch.Tensor | int | None = None, top_p: torch.Tensor | float | None = None,
                  min_p: torch.Tensor | float | None = None) -> tuple:
    """A token for each row of ``logits`` [rows, vocab] (fp16, bf16 or fp32;
    rows may lie apart; vocab up to 2^18) from one random number in [0, 1) a
    row, ``uniform`` fp32 [rows]. Returns ``(tokens, logprobs)``, int64 and fp32
    [rows].

    With T the row's temperature, w_i = exp((l_i - max l) / T). Tokens rank by
    logit, the lower index first. Kept are those of rank below ``top_k`` (0 or
    less: all); those before which less than ``top_p`` of top_k's sum of w ranks
    (1 or more: all); those with w_i >= ``min_p``; and always the first. The
    token is the first, by index, whose running sum of kept w exceeds uniform
    times their sum; its logprob is that of this draw. A temperature of 0 (or
    less) takes the largest logit, with logprob 0. NaN counts as -inf; a row
    without a logit above -inf gives -1 and NaN. A ``uniform`` below 0, or NaN,
    counts as 0; from 1 on it takes the last token kept. (Logits further below the
    largest than fp32's largest number weigh nothing, whatever the temperature.) The
    same inputs give the same tokens: each w is rounded once (2^-31 of itself, or 2^-45) and sums are of
    64-bit integers, whatever their order.

    Each parameter is a number (taken as fp32; top_k as int32), or a tensor of one a
    row of these types."""
    top_k, top_p, min_p = (0 if top_k is None else top_k, 1.0 if top_p is None else top_p,
                           0.0 if min_p is None else min_p)
    if logits.is_cuda:
        return paged._binding().sample_tokens(logits, uniform, temperature, top_k, top_p, min_p)
    inputs = (logits, uniform, temperature, top_k, top_p, min_p)
    if torch.is_grad_enabled() and any(isinstance(x, torch.Tensor) and x.requires_grad for x in inputs):
        raise RuntimeError("a draw has no gradient: an input requires one (call it under torch.no_grad())")
    rows, vocab = logits.shape

    def column(p, dtype):
        return torch.as_tensor(p, dtype=dtype).expand(rows)[:, None]

    heat, p, least = (column(v, torch.float32).double() for v in (temperature, top_p, min_p))
    k = column(top_k, torch.int64)
    x = logits.double()
    x = torch.where(x.isnan(), float("-inf"), x)
    top, order = torch.sort(x, dim=1, descending=True, stable=True)
    largest = top[:, :1]
    w = torch.exp((top - largest) / torch.where(heat > 0, heat, 1.0))
    w = torch.where(torch.isposinf(largest), (top == largest).double(), torch.where(top.isneginf(), 0.0, w))
    rank = torch.arange(vocab)
    kept = (rank < k) | (k <= 0)
    within = torch.where(kept, w, 0.0)
    before = within.cumsum(1) - within
    kept &= (before < p * within.sum(1, keepdim=True)) | ~(p < 1)
    kept &= (w >= least) | ~(least > 0)
    kept = torch.where(heat > 0, kept | (rank == 0), rank == 0)
    w = torch.zeros_like(w).scatter(1, order, torch.where(kept, w, 0.0))
    run_sum = w.cumsum(1)
    total = run_sum[:, -1:]
    u = uniform.double().nan_to_num(0.0).clamp(min=0.0)[:, None]
    token = (run_sum <= u * total).sum(1, keepdim=True)
    token = torch.minimum(token, vocab - 1 - (w.flip(1) > 0).int().argmax(1, keepdim=True))
    logprob = (w.gather(1, token) / total).log().float()
    none = largest.isneginf()
    return torch.where(none, -1, token)[:, 0], torch.where(none, float("nan"), logprob)[:, 0]
