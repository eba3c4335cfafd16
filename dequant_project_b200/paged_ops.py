"""Operators over a key/value cache held in pages: what takes prompts and
batches of different lengths through the decoder's attention.

A cache is two pools ``k_pages``, ``v_pages`` [pages, kv heads, page size, D]
(fp16 or bf16; D 64 or 128; page size 16 to 256, a power of two) and, per
sequence, a row of page numbers in ``block_table``: position t lies in page
``block_table[b, t // page_size]`` at place ``t % page_size``. The pools may be
strided views (of one allocation for keys and values, say) as long as both have
the same strides and D is contiguous.

Forward only: an input that requires a gradient is refused while gradients are
recorded (``torch.no_grad()`` allows it). ``rope_paged_append`` writes the pages
in place.

CUDA tensors go through the sm_100a kernels of libdequant_b200.so on torch's
current stream (checked and called by the native binding,
``binding/paged_binding.cpp``); if either is missing these calls raise. CPU tensors take
the same formulas in torch: that branch exists for the host-logic tests and is
never taken for a CUDA tensor.

The reference has none of this; it models the cache's bytes
(KrishnaI2424/Dequant_Project ``dequant/byte_model.py:214-219``).
"""

from __future__ import annotations

import ctypes
import math

import torch

from dequant_project_b200 import _native

_bound = None


def _binding():
    """The native binding, bound to the library once."""
    global _bound
    if _bound is None:
        lib = _native.lib()
        try:
            from dequant_project_b200 import _paged_binding
        except ImportError as exc:
            raise ImportError(f"_paged_binding.so is not built, or not for this torch and Python ({exc}). "
                              "Build it once with:\n    python -m dequant_project_b200.build") from exc
        if _paged_binding.built_for != torch.__version__:
            raise ImportError(f"_paged_binding.so is built for torch {_paged_binding.built_for}, this is "
                              f"{torch.__version__}. Build it again with:\n    python -m dequant_project_b200.build")
        _paged_binding.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in (
            "dqg_last_error", "dqg_rope_paged_append", "dqg_paged_attention_workspace",
            "dqg_paged_attention", "dqg_prompt_attention_workspace", "dqg_prompt_attention",
            "dqg_shared_prefix_workspace", "dqg_shared_prefix_attention")))
        _bound = _paged_binding
    return _bound


def _forward_only(*inputs) -> None:
    """The binding's refusal, for CPU tensors."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs):
        raise RuntimeError("the paged operators are forward only: an input requires a gradient "
                           "(call them under torch.no_grad())")


# ------------------------------------------------------------------- append
def rope_scaled_tables(head_dim: int, theta: float, positions: int, device, *, rotary_dim: int | None = None,
                       scaling: dict | None = None) -> tuple:
    """cos/sin [positions, rotary_dim / 2] (fp32) for ``rope_paged_append``.

    ``rotary_dim`` (default: the whole head) is the part that rotates.
    ``scaling`` stretches the frequencies for long contexts:
    ``{"type": "linear", "factor": f}`` divides every frequency by f;
    ``{"type": "dynamic", "factor": f, "original": n}`` raises theta so that
    ``positions`` fit where n did; ``{"type": "banded", "factor": f,
    "original": n, "low": a, "high": b}`` keeps frequencies that turn more than
    b times within the original length n, divides by f those that turn less
    than a times, and blends linearly between. Angles are formed in 64 bits."""
    r = head_dim if rotary_dim is None else rotary_dim
    if r % 2 or not 2 <= r <= head_dim:
        raise ValueError(f"rotary_dim must be even and in [2, {head_dim}], got {r}")
    s = scaling or {"type": "none"}
    kind = s.get("type")
    if kind not in ("none", "linear", "dynamic", "banded"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    if kind != "none" and not s["factor"] >= 1.0:
        raise ValueError(f"the scaling factor must be at least 1, got {s['factor']}")
    if kind == "dynamic" and positions > s["original"]:
        if r <= 2:
            raise ValueError("dynamic scaling needs a rotary_dim above 2")
        theta = theta * (s["factor"] * positions / s["original"] - (s["factor"] - 1.0)) ** (r / (r - 2))
    freq = theta ** (-torch.arange(0, r, 2, dtype=torch.float64, device=device) / r)
    if kind == "linear":
        freq = freq / s["factor"]
    elif kind == "banded":
        if not s["high"] > s["low"] > 0:
            raise ValueError("banded scaling needs 0 < low < high")
        turns = s["original"] * freq / (2 * math.pi)
        keep = ((turns - s["low"]) / (s["high"] - s["low"])).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / s["factor"])
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq[None, :]
    return angle.cos().float(), angle.sin().float()


def rope_paged_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                      slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, n_q_heads: int, *,
                      interleaved: bool = False, q_norm: torch.Tensor | None = None,
                      k_norm: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """Norm (optional), rotate and store a batch of tokens: ``qkv``
    [T, (Hq + 2 Hkv) D] -> rotated queries [T, Hq, D]; keys and values are
    written to their pages.

    ``cos``/``sin`` are fp32 [n_positions, R / 2]; token t takes row
    ``positions[t]`` (int64) and rotates the first R values of each query and
    key head: pairs (i, i + R/2), or (2i, 2i + 1) with ``interleaved``.
    ``slots`` (int64 [T]) is page * page_size + place, negative for a token that
    is not stored; no two tokens may share one. ``q_norm``/``k_norm`` [D]:
    x * rsqrt(mean(x^2) + eps) * w per head before the rotation. fp32 math, one
    rounding."""
    if not qkv.is_cuda:
        _forward_only(qkv, cos, sin, k_pages, v_pages, q_norm, k_norm)
        t = qkv.shape[0]
        hkv, page, d = k_pages.shape[1:]
        x = qkv.float().view(t, n_q_heads + 2 * hkv, d)
        q, k, v = x[:, :n_q_heads], x[:, n_q_heads:n_q_heads + hkv], x[:, n_q_heads + hkv:]

        def turn(h, w):
            if w is not None:
                h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * w.float()
            n = cos.shape[1]
            c, s = cos[positions][:, None], sin[positions][:, None]
            a, b = ((h[..., 0:2 * n:2], h[..., 1:2 * n:2]) if interleaved
                    else (h[..., :n], h[..., n:2 * n]))
            lo, hi = a * c - b * s, b * c + a * s
            part = torch.stack([lo, hi], -1).flatten(-2) if interleaved else torch.cat([lo, hi], -1)
            return torch.cat([part, h[..., 2 * n:]], -1).to(qkv.dtype)

        kept = slots >= 0
        at = (slots[kept] // page, slice(None), slots[kept] % page)
        k_pages[at] = turn(k, k_norm)[kept]
        v_pages[at] = v.to(qkv.dtype)[kept]
        return turn(q, q_norm)
    return _binding().rope_paged_append(qkv, cos, sin, positions, slots, k_pages, v_pages, n_q_heads,
                                        interleaved, q_norm, k_norm, eps)


# ---------------------------------------------------------------- attention
def _rows(pages: torch.Tensor, table: torch.Tensor, n: int) -> torch.Tensor:
    """fp32 [kv heads, n, D]: the first n positions that a table row lists."""
    page = pages.shape[2]
    got = pages[table[:-(-n // page)].long()].float()
    return got.transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :n]


def _cpu_attention(q, k, v, ends, scale):
    """q [rows, Hq, D] fp32 over k, v [Hkv, n, D]; row r sees the first
    ends[r] keys (zeros where that is none)."""
    rows, hq, d = q.shape
    hkv, n, _ = k.shape
    if n == 0:
        return torch.zeros_like(q)
    s = torch.einsum("rkgd,ktd->rkgt", q.view(rows, hkv, hq // hkv, d), k) * scale
    seen = (torch.arange(n)[None] < ends[:, None])[:, None, None]
    s = s.masked_fill(~seen, float("-inf"))
    p = torch.softmax(s, -1).masked_fill(~seen, 0.0)
    fine = torch.isfinite(v)
    out = torch.einsum("rkgt,ktd->rkgd", p, torch.where(fine, v, 0.0))
    # A weight of zero times an infinity is not zero: rows take the non-finite
    # values that they see, and no others.
    for t in torch.nonzero(~fine.all(-1).all(0))[:, 0].tolist():
        x = torch.where(fine[:, t], 0.0, v[:, t])[None, :, None]
        out = out + torch.where(seen[..., t, None], x, 0.0)
    return out.reshape(rows, hq, d)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, *, scale: float | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """One query token per sequence over its cached positions.

    q [B, Hq, D] (strides free, D contiguous), block_table int32
    [B, pages per sequence], kv_lens int32 [B]. Returns [B, Hq, D]; zeros for a
    sequence without positions. The lengths stay on the device: a captured call
    serves other lengths. ``workspace`` (``paged_attention_workspace``) keeps the
    call from taking scratch memory of its own; calls that share one must not
    overlap."""
    if q.is_cuda:
        return _binding().paged_attention(q, k_pages, v_pages, block_table, kv_lens, scale, workspace)
    _forward_only(q, k_pages, v_pages)
    b, _, d = q.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = [_cpu_attention(q[i:i + 1].float(), _rows(k_pages, block_table[i], int(kv_lens[i])),
                          _rows(v_pages, block_table[i], int(kv_lens[i])), kv_lens[i:i + 1], scale)
           for i in range(b)]
    return torch.cat(out).to(q.dtype) if out else torch.empty_like(q)


def paged_attention_workspace(n_seqs: int, n_q_heads: int, n_kv_heads: int, head_dim: int, device) -> torch.Tensor:
    """Scratch memory for ``paged_attention`` calls of these sizes and any lengths."""
    return shared_prefix_workspace(n_seqs, n_q_heads, n_kv_heads, head_dim, 0, device)


def prompt_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                     q_starts: torch.Tensor, kv_lens: torch.Tensor, *, causal: bool = True,
                     scale: float | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Packed prompts (or chunks at their ends) over their cached positions.

    q [T, Hq, D] holds the new tokens of all sequences one after the other:
    sequence b has rows ``q_starts[b]`` to ``q_starts[b + 1] - 1`` (int32
    [B + 1], from 0 to T), and they are the newest of its ``kv_lens[b]`` cached
    positions (so they were stored first). Row i of q_len sees the keys before
    kv_len - q_len + i + 1 (all kv_len unless ``causal``); a row that sees none
    gives zeros, and what a row does not see does not matter to it, non-finite
    values included. Rows outside every sequence are undefined in the result.
    Returns [T, Hq, D]. Table, lengths, scale and workspace
    (``prompt_attention_workspace``) as ``paged_attention``."""
    if q.is_cuda:
        return _binding().prompt_attention(q, k_pages, v_pages, block_table, q_starts, kv_lens, causal, scale,
                                           workspace)
    _forward_only(q, k_pages, v_pages)
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    out = torch.zeros_like(q)
    for i in range(kv_lens.shape[0]):
        lo, hi, n = int(q_starts[i]), int(q_starts[i + 1]), int(kv_lens[i])
        ends = n - (hi - lo) + torch.arange(hi - lo) + 1 if causal else torch.full((hi - lo,), n)
        out[lo:hi] = _cpu_attention(q[lo:hi].float(), _rows(k_pages, block_table[i], n),
                                    _rows(v_pages, block_table[i], n), ends, scale).to(q.dtype)
    return out


def _bytes(device, call, *args) -> torch.Tensor:
    n = ctypes.c_uint64(0)
    with torch.cuda.device(device):
        _native.check(call(*args, ctypes.byref(n)))
        return torch.empty(max(16, n.value), dtype=torch.uint8, device=device)


def prompt_attention_workspace(head_dim: int, device) -> torch.Tensor:
    """Scratch memory for ``prompt_attention`` calls of any batch and lengths."""
    return _bytes(device, _native.lib().dqg_prompt_attention_workspace, head_dim)


def shared_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                            prefix_table: torch.Tensor, prefix_len: int, block_table: torch.Tensor,
                            kv_lens: torch.Tensor, *, scale: float | None = None,
                            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_attention`` for a batch whose sequences share their first
    ``prefix_len`` positions (a system prompt, a document that is sampled from
    many times): those lie in the pages of ``prefix_table`` (int32
    [prefix pages]) and are read once for many sequences (once or twice for a
    small batch, once for every 256 / (Hq / Hkv) of a larger one); ``block_table`` and
    ``kv_lens`` are each sequence's own positions after them (none is fine).
    ``workspace``: ``shared_prefix_workspace``."""
    if q.is_cuda:
        return _binding().shared_prefix_attention(q, k_pages, v_pages, prefix_table, prefix_len, block_table,
                                                  kv_lens, scale, workspace)
    _forward_only(q, k_pages, v_pages)
    b, _, d = q.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = []
    for i in range(b):
        n = int(kv_lens[i])
        k, v = (torch.cat([_rows(p, prefix_table, prefix_len), _rows(p, block_table[i], n)], 1)
                for p in (k_pages, v_pages))
        out.append(_cpu_attention(q[i:i + 1].float(), k, v, torch.tensor([prefix_len + n]), scale))
    return torch.cat(out).to(q.dtype) if out else torch.empty_like(q)


def shared_prefix_workspace(n_seqs: int, n_q_heads: int, n_kv_heads: int, head_dim: int, prefix_len: int,
                            device) -> torch.Tensor:
    """Scratch memory for ``shared_prefix_attention`` calls of these sizes."""
    return _bytes(device, _native.lib().dqg_shared_prefix_workspace, n_seqs, n_q_heads, n_kv_heads, head_dim,
                  prefix_len)
