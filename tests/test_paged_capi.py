"""Paged-cache entry points of the C ABI: bad arguments are rejected, with a
message, before anything touches the GPU (runs on CPU-only hosts)."""

from __future__ import annotations

import ctypes

import pytest

from dequant_project_b200 import _native


def pool(**kw):
    a = dict(k=1 << 20, v=1 << 21, n_pages=4, n_kv_heads=2, page_size=16, head_dim=128, page_stride=4096,
             head_stride=2048, row_stride=128, dtype=0)
    a.update(kw)
    return _native.PagedKV(*a.values())


POOLS = [
    (dict(k=None), 1, "k_pages must not be null"),
    (dict(v=(1 << 21) + 8), 1, "v_pages must be 16-byte aligned"),
    (dict(dtype=2), 1, "dtype must be"),
    (dict(head_dim=96), 2, "head_dim 64 and 128, got 96"),
    (dict(page_size=8), 2, "page_size must be 16"),
    (dict(page_size=48), 2, "page_size must be 16"),
    (dict(page_size=512), 2, "page_size must be 16"),
    (dict(n_kv_heads=0), 1, "n_kv_heads must be in"),
    (dict(n_pages=0), 1, "n_pages must be in"),
    (dict(page_stride=4100), 1, "page stride must be a positive multiple of 8"),
    (dict(head_stride=0), 1, "head stride must be a positive multiple of 8"),
    (dict(row_stride=64), 1, "rows overlap"),
]


def rejected(rc, code, msg):
    assert rc == code
    assert msg in _native.lib().dqg_last_error().decode()


def append(kv=None, **kw):
    a = dict(qkv=16, T=3, stride=1024, hq=4, cos=16, sin=16, n=8, rot=128, inter=0, pos=16, slots=16, qn=None,
             kn=None, eps=1e-5)
    a.update(kw)
    return _native.lib().dqg_rope_paged_append(*a.values(), pool() if kv is None else kv, 16, None)


def decode(kv=None, **kw):
    a = dict(q=16, qs=512, qh=128, n=2, hq=4)
    b = dict(table=16, width=3, stride=3, lens=16, scale=0.1, out=16, ws=16, bytes=1 << 40)
    for k, v in kw.items():
        (a if k in a else b)[k] = v
    return _native.lib().dqg_paged_attention(*a.values(), pool() if kv is None else kv, *b.values(), None)


def prompt(kv=None, **kw):
    a = dict(q=16, qs=512, qh=128, T=5, hq=4)
    b = dict(table=16, width=3, stride=3, starts=16, lens=16, n=2, causal=1, scale=0.1, out=16, ws=16,
             bytes=1 << 40)
    for k, v in kw.items():
        (a if k in a else b)[k] = v
    return _native.lib().dqg_prompt_attention(*a.values(), pool() if kv is None else kv, *b.values(), None)


@pytest.mark.parametrize("call", [append, decode, prompt], ids=lambda f: f.__name__)
@pytest.mark.parametrize("kw,code,msg", POOLS, ids=lambda v: str(v))
def test_pools(call, kw, code, msg):
    rejected(call(pool(**kw)), code, msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=-1), "T=-1 out of range"),
    (dict(stride=1000), "row stride"),
    (dict(stride=1028), "row stride"),
    (dict(hq=3), "must give 1..128 query heads"),
    (dict(rot=0), "rotary_dim must be even"),
    (dict(rot=7), "rotary_dim must be even"),
    (dict(rot=130), "rotary_dim must be even"),
    (dict(n=0), "at least one position"),
    (dict(qn=16), "given together"),
    (dict(eps=-1.0), "eps must be non-negative"),
    (dict(eps=float("nan")), "eps must be non-negative"),
    (dict(qkv=8), "qkv must be 16-byte aligned"),
    (dict(pos=12), "positions must be 8-byte aligned"),
    (dict(slots=None), "slots must not be null"),
    (dict(qn=16, kn=8), "k_norm must be 16-byte aligned"),
], ids=lambda v: str(v))
def test_append(kw, msg):
    rejected(append(**kw), 1, msg)


ATTENTION = [
    (dict(q=None), "q must not be null"),
    (dict(q=24), "q must be 16-byte aligned"),
    (dict(qh=64), "q's strides"),
    (dict(qs=516), "q's strides"),
    (dict(hq=5), "must give 1..128 query heads"),
    (dict(hq=512), "must give 1..128 query heads"),
    (dict(table=None), "block_table must not be null"),
    (dict(width=0), "at least one page"),
    (dict(stride=2), "at least one page"),
    (dict(lens=6), "kv_lens must be 4-byte aligned"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=float("inf")), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
    (dict(out=8), "out must be 16-byte aligned"),
]


@pytest.mark.parametrize("call", [decode, prompt], ids=lambda f: f.__name__)
@pytest.mark.parametrize("kw,msg", ATTENTION, ids=lambda v: str(v))
def test_attention(call, kw, msg):
    rejected(call(**kw), 1, msg)


def test_counts_and_empty_calls():
    rejected(decode(n=-1), 1, "n_seqs=-1 out of range")
    rejected(prompt(n=-1), 1, "n_seqs=-1 out of range")
    rejected(prompt(T=1 << 40), 1, "out of range")
    rejected(prompt(starts=None), 1, "q_starts must not be null")
    # Nothing to do: nothing is launched, nothing else is looked at.
    assert append(T=0) == 0 and decode(n=0) == 0 and prompt(T=0) == 0 and prompt(n=0) == 0


def test_workspace_queries():
    lib, n = _native.lib(), ctypes.c_uint64(0)
    rejected(lib.dqg_prompt_attention_workspace(96, ctypes.byref(n)), 2, "head_dim 64 and 128")
    rejected(lib.dqg_paged_attention_workspace(2, 4, 3, 128, ctypes.byref(n)), 1, "query heads per KV head")
    rejected(lib.dqg_shared_prefix_workspace(2, 4, 2, 128, -1, ctypes.byref(n)), 1, "prefix_len=-1")
    rejected(lib.dqg_shared_prefix_workspace(2, 4, 2, 128, 8, None), 1, "bytes must not be null")


def test_struct_layout():
    """dqg_paged_kv as ctypes lays it out: two pointers, seven 64-bit counts, a
    32-bit type."""
    assert ctypes.sizeof(_native.PagedKV) == 2 * 8 + 7 * 8 + 8
    assert _native.PagedKV.dtype.offset == 72
