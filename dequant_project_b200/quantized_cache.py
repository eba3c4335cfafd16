"""Operators over a key/value cache held in 8 bits: half the bytes that a
decode step of ``paged_ops`` reads, and twice the positions in the same memory.

A ``QuantizedCache`` is pages of codes (int8 or e4m3) with an fp32 scale for
every ``block`` positions (16, 32 or 64, at most a page) of each KV head; a
value is code * scale. A block is quantised once, when its last position is
stored: until then its rows wait in 16 bits in the sequence's *open block*, a
row of the pools ``k_open``/``v_open`` that the caller gives each sequence
(``open_slots``, int32 [B]; no two live sequences share one). So what the cache
holds does not depend on how a prompt was cut into calls, no value is rounded
twice, and the newest positions are exact. A block that holds a value that is
not finite reads as NaN.

The pages' table, lengths and sizes are those of ``paged_ops``; lengths, tables
and slots are read on the device, so captured calls serve others. A page, slot,
position or row start out of range is left out and reported by
``_native.device_status``. Forward only, as ``paged_ops``.

CUDA tensors go through the sm_100a kernels of libdequant_b200.so on torch's
current stream (``binding/paged_binding.cpp``); if it is missing these calls
raise. CPU tensors take the same formulas in torch: that branch exists for the
host-logic tests and is never taken where a cache or its queries are on a GPU.

The reference has none of this; it models the cache's bytes
(KrishnaI2424/Dequant_Project ``dequant/byte_model.py:214-219``).
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from dequant_project_b200 import _native
from dequant_project_b200 import paged_ops as paged

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LEAST_SCALE = 2.0 ** -126


class QuantizedCache(NamedTuple):
    """``k``, ``v``: codes [pages, kv heads, page size, D], int8 or
    float8_e4m3fn. ``k_scale``, ``v_scale``: fp32 [pages, kv heads, page size /
    block]. ``k_open``, ``v_open``: [slots, kv heads, block, D], fp16 or bf16:
    the type of queries and outputs. The two of a pair have the same strides;
    D, a page's scales and an open block are contiguous."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    k_open: torch.Tensor
    v_open: torch.Tensor

    @classmethod
    def empty(cls, n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, n_slots: int, *, block: int = 16,
              codes: torch.dtype = torch.int8, dtype: torch.dtype = torch.float16, device="cuda") -> "QuantizedCache":
        """A cache of zeros for up to ``n_slots`` sequences."""
        if codes not in MOST:
            raise ValueError(f"codes must be int8 or float8_e4m3fn, got {codes}")
        if block not in (16, 32, 64) or page_size % block:
            raise ValueError(f"block must be 16, 32 or 64 and divide the page of {page_size}, got {block}")
        pages = [torch.zeros((n_pages, n_kv_heads, page_size, head_dim), dtype=torch.uint8, device=device).view(codes)
                 for _ in range(2)]
        scales = [torch.zeros((n_pages, n_kv_heads, page_size // block), device=device) for _ in range(2)]
        opens = [torch.zeros((n_slots, n_kv_heads, block, head_dim), dtype=dtype, device=device) for _ in range(2)]
        return cls(*pages, *scales, *opens)

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def block(self) -> int:
        return self.k_open.shape[2]


# ------------------------------------------------------------------- append
def quantize_block(x: torch.Tensor, codes: torch.dtype) -> tuple:
    """Codes of a block's values [..., block, D] and their scale [...], as the
    kernel forms them (on the CPU, for the host branch and its tests)."""
    x = x.float()
    most = x.abs().amax((-1, -2))
    scale = torch.where(torch.isfinite(most), (most / MOST[codes]).clamp(min=LEAST_SCALE), float("nan"))
    # (L x) / max |x|, the product exact: x / scale without the scale's rounding
    # (large values by 2^-64 of themselves: bf16's largest times L is no number).
    less = torch.where(most > 1e30, 2.0 ** -64, 1.0)
    x, most = x * less[..., None, None], most * less
    tiny = (scale <= LEAST_SCALE)[..., None, None]
    y = torch.where(tiny, x * 2.0 ** 126, x * MOST[codes] / most[..., None, None])
    y = torch.where(torch.isfinite(scale)[..., None, None], y, 0.0)
    if codes == torch.int8:
        return torch.round(y).clamp(-127, 127).to(torch.int8), scale
    return y.clamp(-448, 448).to(codes), scale


def _rows(cache: QuantizedCache, which: int, table: torch.Tensor, slot: int, n: int) -> torch.Tensor:
    """fp32 [kv heads, n, D]: a sequence's first n positions."""
    codes, scale, opened = cache[which], cache[2 + which], cache[4 + which]
    page, block = cache.page_size, cache.block
    done = n - n % block
    t = torch.arange(done)
    at = table.long()[t // page]
    x = codes.float()[at, :, t % page] * scale[at, :, t % page // block][..., None]
    return torch.cat([x.transpose(0, 1), opened[slot, :, :n - done].float()], 1)


def _put(cache: QuantizedCache, which: int, table: torch.Tensor, slot: int, end: int, new: torch.Tensor) -> None:
    """Store ``new`` [kv heads, n, D] as the newest of ``end`` positions."""
    codes, scale, opened = cache[which], cache[2 + which], cache[4 + which]
    page, block = cache.page_size, cache.block
    start = end - new.shape[1]
    base = start - start % block
    rows = torch.cat([opened[slot, :, :start - base], new], 1)
    while base + block <= end:
        at, part = int(table[base // page]), base % page
        c, s = quantize_block(rows[:, :block], codes.dtype)
        codes.view(torch.uint8)[at, :, part:part + block] = c.view(torch.uint8)
        scale[at, :, part // block] = s
        rows, base = rows[:, block:], base + block
    opened[slot, :, :end - base] = rows


def rope_quantized_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                          cache: QuantizedCache, block_table: torch.Tensor, open_slots: torch.Tensor,
                          q_starts: torch.Tensor, kv_lens: torch.Tensor, n_q_heads: int, *,
                          interleaved: bool = False, q_norm: torch.Tensor | None = None,
                          k_norm: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """``paged_ops.rope_paged_append`` into an 8-bit cache: norm (optional),
    rotate and store a batch of tokens, ``qkv`` [T, (Hq + 2 Hkv) D] -> rotated
    queries [T, Hq, D].

    Sequence b's new tokens are rows ``q_starts[b]`` to ``q_starts[b + 1] - 1``
    (int32 [B + 1], ascending), the newest of its ``kv_lens[b]`` positions,
    these included; they go to the pages of its row of ``block_table`` (int32
    [B, pages]) and to its open block. Rows behind the last sequence are rotated
    and not stored. Keys and values are rounded to the 16-bit type first, as a
    16-bit cache holds them. Everything else as ``rope_paged_append``."""
    if qkv.is_cuda or cache.k.is_cuda:
        return paged._binding().rope_quantized_append(qkv, cos, sin, positions, *cache, block_table, open_slots,
                                                      q_starts, kv_lens, n_q_heads, interleaved, q_norm, k_norm, eps)
    paged._forward_only(qkv, cos, sin, *cache, q_norm, k_norm)
    t, hkv, d = qkv.shape[0], cache.k.shape[1], cache.k.shape[3]
    # Rotated keys and rounded values, from pages of one position each.
    k, v = (torch.zeros((t, hkv, 1, d), dtype=qkv.dtype) for _ in range(2))
    q = paged.rope_paged_append(qkv, cos, sin, positions, torch.arange(t), k, v, n_q_heads, interleaved=interleaved,
                                q_norm=q_norm, k_norm=k_norm, eps=eps)
    for b in range(kv_lens.shape[0]):
        lo, hi = int(q_starts[b]), int(q_starts[b + 1])
        if hi > lo:
            for which, x in ((0, k), (1, v)):
                _put(cache, which, block_table[b], int(open_slots[b]), int(kv_lens[b]), x[lo:hi, :, 0].transpose(0, 1))
    return q


# ---------------------------------------------------------------- attention
def quantized_attention(q: torch.Tensor, cache: QuantizedCache, block_table: torch.Tensor, open_slots: torch.Tensor,
                        kv_lens: torch.Tensor, *, scale: float | None = None,
                        workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_ops.paged_attention`` over an 8-bit cache: one query token per
    sequence, q [B, Hq, D] (strides free, D contiguous) -> [B, Hq, D]; zeros for
    a sequence without positions. Codes enter the products exactly (int8 ones
    beside queries to 2^-23 of their head's largest value), scales in fp32.
    ``workspace``: ``quantized_attention_workspace``; calls that share one must not
    overlap."""
    if q.is_cuda or cache.k.is_cuda:
        return paged._binding().quantized_attention(q, *cache, block_table, open_slots, kv_lens, scale, workspace)
    paged._forward_only(q, *cache)
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    out = [paged._cpu_attention(q[b:b + 1].float(), *(_rows(cache, w, block_table[b], int(open_slots[b]), int(n))
                                                      for w in (0, 1)), kv_lens[b:b + 1], scale)
           for b, n in enumerate(kv_lens)]
    return torch.cat(out).to(q.dtype) if out else torch.empty_like(q)


def quantized_attention_workspace(n_seqs: int, n_q_heads: int, n_kv_heads: int, head_dim: int,
                                  device) -> torch.Tensor:
    """Scratch memory for ``quantized_attention`` calls of these sizes and any lengths."""
    return paged._bytes(device, _native.lib().dqg_quantized_attention_workspace, n_seqs, n_q_heads, n_kv_heads,
                        head_dim)


def expanded_pages(cache: QuantizedCache, block_table: torch.Tensor, open_slots: torch.Tensor, kv_lens: torch.Tensor,
                   n_pages: int) -> tuple:
    """The sequences' positions as 16-bit pages that ``paged_ops`` reads:
    ``(k_pages, v_pages, table)``, pools of ``n_pages`` pages and a table as
    ``block_table``. One sequence's pages follow the other's; each value is
    rounded once to the 16-bit type, and places behind a sequence's end are
    zeros; the table's entries behind a sequence's pages are undefined. ``n_pages``
    is the number that the sequences take (sum of ceil(len / page size)) or more;
    what has no room is left out and reported, pages that nothing takes are
    undefined."""
    if cache.k.is_cuda:
        return paged._binding().expand_pages(*cache, block_table, open_slots, kv_lens, n_pages)
    paged._forward_only(*cache)
    at, page = 0, cache.page_size
    k, v = (torch.empty((n_pages, cache.k.shape[1], page, cache.k.shape[3]), dtype=cache.k_open.dtype) for _ in range(2))
    table = torch.full_like(block_table, -1)
    for b, n in enumerate(kv_lens.tolist()):
        taken = -(-n // page)
        table[b, :taken] = torch.arange(at, at + taken)
        for which, out in ((0, k), (1, v)):
            x = _rows(cache, which, block_table[b], int(open_slots[b]), n)
            x = torch.nn.functional.pad(x, (0, 0, 0, taken * page - n))
            out[at:at + taken] = x.unflatten(1, (taken, page)).transpose(0, 1).to(out.dtype)
        at += taken
    return k, v, table


def quantized_prompt_attention(q: torch.Tensor, cache: QuantizedCache, block_table: torch.Tensor,
                               open_slots: torch.Tensor, q_starts: torch.Tensor, kv_lens: torch.Tensor, n_pages: int,
                               *, causal: bool = True, scale: float | None = None,
                               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_ops.prompt_attention`` over an 8-bit cache, whose positions are
    first expanded once to 16-bit pages (as ``expanded_pages``, which says what
    ``n_pages`` is; but keys stay codes and values codes times a power of two, exact
    in 16 bits but for the smallest in fp16, off by up to 2^-24; and the rest of the
    scales goes to the scores and weights in fp32).
    ``workspace``: ``quantized_prompt_workspace``, mostly n_pages * 4 * Hkv *
    page size * D bytes; calls that share one must not overlap. Everything else
    as ``prompt_attention``."""
    if q.is_cuda or cache.k.is_cuda:
        return paged._binding().quantized_prompt_attention(q, *cache, block_table, open_slots, q_starts, kv_lens,
                                                           n_pages, causal, scale, workspace)
    paged._forward_only(q, *cache)
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    out = torch.zeros_like(q)
    for b in range(kv_lens.shape[0]):
        lo, hi, n = int(q_starts[b]), int(q_starts[b + 1]), int(kv_lens[b])
        ends = n - (hi - lo) + torch.arange(hi - lo) + 1 if causal else torch.full((hi - lo,), n)
        k, v = (_rows(cache, w, block_table[b], int(open_slots[b]), n) for w in (0, 1))
        out[lo:hi] = paged._cpu_attention(q[lo:hi].float(), k, v, ends, scale).to(q.dtype)
    return out


def quantized_prompt_workspace(cache: QuantizedCache, n_seqs: int, table_width: int, n_pages: int) -> torch.Tensor:
    """Scratch memory for ``quantized_prompt_attention`` calls of these sizes
    (``table_width``: block_table's) and any lengths."""
    kv = _native.QuantizedKV(*(t.data_ptr() for t in cache), *cache.k.shape, cache.block, cache.k_open.shape[0],
                             *cache.k.stride()[:3], *cache.k_scale.stride()[:2], *cache.k_open.stride()[:2],
                             int(cache.k.dtype == torch.float8_e4m3fn), int(cache.k_open.dtype == torch.bfloat16))
    return paged._bytes(cache.k.device, _native.lib().dqg_quantized_prompt_workspace, ctypes.byref(kv), n_seqs,
                        table_width, n_pages)
