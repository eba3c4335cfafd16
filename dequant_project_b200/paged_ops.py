"""Operators over a key/value cache held in pages: what takes prompts and
batches of different lengths through the decoder's attention.

A cache is two pools ``k_pages``, ``v_pages`` [pages, kv heads, page size, D]
(fp16 or bf16; D 64 or 128; page size 16 to 256, a power of two) and, per
sequence, a row of page numbers in ``block_table``: position t lies in page
``block_table[b, t // page_size]`` at place ``t % page_size``. The pools may be
strided views (of one allocation for keys and values, say) as long as both have
the same strides and D is contiguous.

CUDA tensors go through the sm_100a kernels of libdequant_b200.so on torch's
current stream; if the library is missing these calls raise. CPU tensors take
the same formulas in torch: that branch exists for the host-logic tests and is
never taken for a CUDA tensor.

The reference has none of this; it models the cache's bytes
(KrishnaI2424/Dequant_Project ``dequant/byte_model.py:214-219``).
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import math

import torch

from dequant_project_b200 import _native

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}


def _pools(k: torch.Tensor, v: torch.Tensor, name: str, t: torch.Tensor) -> tuple:
    """The C description of the pools and their device, with the checks that
    need tensors; ``t`` (``name`` in messages) must have their type and device."""
    dtype, shape, strides, dev = k.dtype, k.shape, k.stride(), t.get_device()
    if (dtype not in _DTYPES or len(shape) != 4 or strides[3] != 1 or v.stride() != strides or v.shape != shape
            or v.dtype is not dtype or t.dtype is not dtype or k.get_device() != dev or v.get_device() != dev):
        if dtype not in _DTYPES:
            raise RuntimeError(f"pages must be float16 or bfloat16, got {dtype}")
        if len(shape) != 4:
            raise RuntimeError("pages must be [pages, kv heads, page size, head dim]")
        if v.stride() != strides or v.shape != shape or v.dtype is not dtype or strides[3] != 1:
            raise RuntimeError("k_pages and v_pages must have one shape, type and strides, with the "
                               "head dimension contiguous")
        if v.device != k.device:
            raise RuntimeError("k_pages and v_pages must be on the same device")
        raise RuntimeError(f"{name} must be {dtype} on {k.device}, as the pages are")
    return _native.PagedKV(k.data_ptr(), v.data_ptr(), *shape, strides[0], strides[1], strides[2],
                           _DTYPES[dtype]), dev


def _ints(name: str, t: torch.Tensor, dtype, dims: int, dev: int) -> None:
    """An integer tensor whose last dimension is contiguous."""
    if t.dtype is not dtype or t.dim() != dims or t.get_device() != dev or t.stride()[-1] != 1:
        raise RuntimeError(f"{name} must be a contiguous {dims}-dimensional {dtype} tensor on cuda:{dev}")


def _on(dev: int):
    """The device as the current one, for callers that have another current."""
    return _SAME if dev == torch._C._cuda_getDevice() else torch.cuda.device(dev)


def _index(device) -> int:
    index = torch.device(device).index
    return torch.cuda.current_device() if index is None else index


_SAME = contextlib.nullcontext()


_stream = torch._C._cuda_getCurrentRawStream if torch.cuda._is_compiled() else None


@functools.lru_cache(maxsize=None)
def _prompt_bytes(device_index: int, head_dim: int) -> int:
    n = ctypes.c_uint64(0)
    _native.check(_native.lib().dqg_prompt_attention_workspace(head_dim, ctypes.byref(n)))
    return int(n.value)


@functools.lru_cache(maxsize=1024)
def _prefix_bytes(device_index: int, n_seqs: int, hq: int, hkv: int, head_dim: int, prefix_len: int) -> int:
    n = ctypes.c_uint64(0)
    _native.check(_native.lib().dqg_shared_prefix_workspace(n_seqs, hq, hkv, head_dim, prefix_len,
                                                            ctypes.byref(n)))
    return int(n.value)


def _workspace(given: torch.Tensor | None, need: int, q: torch.Tensor) -> tuple:
    """(tensor, pointer, bytes) of the scratch memory of a call on ``q``."""
    if given is None:
        given = q.new_empty(need, dtype=torch.uint8)
        return given, given.data_ptr(), need
    if given.get_device() != q.get_device() or not given.is_contiguous():
        raise RuntimeError(f"the workspace must be a contiguous tensor on {q.device}")
    return given, given.data_ptr(), given.numel() * given.element_size()


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
    t = qkv.shape[0]
    hkv, page, d = k_pages.shape[1:]
    if not qkv.is_cuda:
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
    kv, dev = _pools(k_pages, v_pages, "qkv", qkv)
    if qkv.dim() != 2 or qkv.shape[1] != (n_q_heads + 2 * hkv) * d or qkv.stride(1) != 1:
        raise RuntimeError(f"qkv must be [T, {(n_q_heads + 2 * hkv) * d}] with contiguous rows")
    shape = cos.shape
    if (cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or len(shape) != 2 or sin.shape != shape
            or cos.get_device() != dev or sin.get_device() != dev
            or not (cos.is_contiguous() and sin.is_contiguous())):
        raise RuntimeError(f"cos and sin must be contiguous float32 [positions, R / 2] on cuda:{dev}")
    _ints("positions", positions, torch.int64, 1, dev)
    _ints("slots", slots, torch.int64, 1, dev)
    if positions.shape[0] != t or slots.shape[0] != t:
        raise RuntimeError(f"positions and slots must hold one entry for each of the {t} tokens")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None and (w.shape != (d,) or w.stride(0) != 1 or w.dtype is not qkv.dtype
                              or w.get_device() != dev):
            raise RuntimeError(f"{name} must hold {d} contiguous {qkv.dtype} weights on cuda:{dev}")
    q = qkv.new_empty((t, n_q_heads, d))
    with _on(dev):
        _native.check(_native.lib().dqg_rope_paged_append(
            qkv.data_ptr(), t, qkv.stride(0) if t > 1 else qkv.shape[1], n_q_heads, cos.data_ptr(),
            sin.data_ptr(), shape[0], 2 * shape[1], interleaved, positions.data_ptr(), slots.data_ptr(),
            None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), eps,
            kv, q.data_ptr(), _stream(dev)))
    return q


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
    return torch.einsum("rkgt,ktd->rkgd", p, v).reshape(rows, hq, d)


def _query(q: torch.Tensor, d: int) -> None:
    if q.dim() != 3 or q.shape[2] != d or q.stride(2) != 1:
        raise RuntimeError(f"q must be [rows, heads, {d}] with the head dimension contiguous")


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
    b, hq, d = q.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if not q.is_cuda:
        out = [_cpu_attention(q[i:i + 1].float(), _rows(k_pages, block_table[i], int(kv_lens[i])),
                              _rows(v_pages, block_table[i], int(kv_lens[i])), kv_lens[i:i + 1], scale)
               for i in range(b)]
        return torch.cat(out).to(q.dtype) if out else torch.empty_like(q)
    kv, dev = _pools(k_pages, v_pages, "q", q)
    _query(q, kv.head_dim)
    _ints("block_table", block_table, torch.int32, 2, dev)
    _ints("kv_lens", kv_lens, torch.int32, 1, dev)
    if block_table.shape[0] != b or kv_lens.shape[0] != b:
        raise RuntimeError(f"block_table and kv_lens must hold one row for each of the {b} sequences")
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    with _on(dev):
        _, ws, size = _workspace(workspace, _prefix_bytes(dev, b, hq, kv.n_kv_heads, d, 0), q)
        _native.check(_native.lib().dqg_paged_attention(
            q.data_ptr(), q.stride(0), q.stride(1), b, hq, kv, block_table.data_ptr(),
            block_table.shape[1], block_table.stride(0) if b > 1 else block_table.shape[1],
            kv_lens.data_ptr(), scale, out.data_ptr(), ws, size, _stream(dev)))
    return out


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
    gives zeros. Rows outside every sequence are undefined in the result.
    Returns [T, Hq, D]. Table, lengths, scale and workspace
    (``prompt_attention_workspace``) as ``paged_attention``."""
    t, hq, d = q.shape
    b = kv_lens.shape[0]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if not q.is_cuda:
        out = torch.zeros_like(q)
        for i in range(b):
            lo, hi, n = int(q_starts[i]), int(q_starts[i + 1]), int(kv_lens[i])
            ends = (n - (hi - lo) + torch.arange(hi - lo) + 1 if causal else torch.full((hi - lo,), n))
            out[lo:hi] = _cpu_attention(q[lo:hi].float(), _rows(k_pages, block_table[i], n),
                                        _rows(v_pages, block_table[i], n), ends, scale).to(q.dtype)
        return out
    kv, dev = _pools(k_pages, v_pages, "q", q)
    _query(q, kv.head_dim)
    _ints("block_table", block_table, torch.int32, 2, dev)
    _ints("q_starts", q_starts, torch.int32, 1, dev)
    _ints("kv_lens", kv_lens, torch.int32, 1, dev)
    if block_table.shape[0] != b or q_starts.shape[0] != b + 1:
        raise RuntimeError(f"block_table and q_starts must hold {b} and {b + 1} rows for {b} sequences")
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    with _on(dev):
        _, ws, size = _workspace(workspace, _prompt_bytes(dev, d), q)
        _native.check(_native.lib().dqg_prompt_attention(
            q.data_ptr(), q.stride(0), q.stride(1), t, hq, kv, block_table.data_ptr(),
            block_table.shape[1], block_table.stride(0) if b > 1 else block_table.shape[1],
            q_starts.data_ptr(), kv_lens.data_ptr(), b, causal, scale, out.data_ptr(), ws, size,
            _stream(dev)))
    return out


def prompt_attention_workspace(head_dim: int, device) -> torch.Tensor:
    """Scratch memory for ``prompt_attention`` calls of any batch and lengths."""
    dev = _index(device)
    with _on(dev):
        return torch.empty(_prompt_bytes(dev, head_dim), dtype=torch.uint8, device=device)


def shared_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                            prefix_table: torch.Tensor, prefix_len: int, block_table: torch.Tensor,
                            kv_lens: torch.Tensor, *, scale: float | None = None,
                            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_attention`` for a batch whose sequences share their first
    ``prefix_len`` positions (a system prompt, a document that is sampled from
    many times): those lie in the pages of ``prefix_table`` (int32
    [prefix pages]) and are read once for the whole batch; ``block_table`` and
    ``kv_lens`` are each sequence's own positions after them (none is fine).
    ``workspace``: ``shared_prefix_workspace``."""
    b, hq, d = q.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if not q.is_cuda:
        out = []
        for i in range(b):
            n = int(kv_lens[i])
            k, v = (torch.cat([_rows(p, prefix_table, prefix_len), _rows(p, block_table[i], n)], 1)
                    for p in (k_pages, v_pages))
            out.append(_cpu_attention(q[i:i + 1].float(), k, v, torch.tensor([prefix_len + n]), scale))
        return torch.cat(out).to(q.dtype) if out else torch.empty_like(q)
    kv, dev = _pools(k_pages, v_pages, "q", q)
    _query(q, kv.head_dim)
    _ints("prefix_table", prefix_table, torch.int32, 1, dev)
    _ints("block_table", block_table, torch.int32, 2, dev)
    _ints("kv_lens", kv_lens, torch.int32, 1, dev)
    if block_table.shape[0] != b or kv_lens.shape[0] != b:
        raise RuntimeError(f"block_table and kv_lens must hold one row for each of the {b} sequences")
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    with _on(dev):
        _, ws, size = _workspace(workspace, _prefix_bytes(dev, b, hq, kv.n_kv_heads, d, prefix_len), q)
        _native.check(_native.lib().dqg_shared_prefix_attention(
            q.data_ptr(), q.stride(0), q.stride(1), b, hq, kv, prefix_table.data_ptr(),
            prefix_table.shape[0], prefix_len, block_table.data_ptr(), block_table.shape[1],
            block_table.stride(0) if b > 1 else block_table.shape[1], kv_lens.data_ptr(), scale,
            out.data_ptr(), ws, size, _stream(dev)))
    return out


def shared_prefix_workspace(n_seqs: int, n_q_heads: int, n_kv_heads: int, head_dim: int, prefix_len: int,
                            device) -> torch.Tensor:
    """Scratch memory for ``shared_prefix_attention`` calls of these sizes."""
    dev = _index(device)
    with _on(dev):
        return torch.empty(_prefix_bytes(dev, n_seqs, n_q_heads, n_kv_heads, head_dim, prefix_len),
                           dtype=torch.uint8, device=device)
