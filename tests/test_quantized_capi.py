"""Entry points of the 8-bit cache and of the token draw in the C ABI: bad
arguments are rejected, with a message, before anything touches the GPU (runs
on CPU-only hosts)."""

from __future__ import annotations

import ctypes

import pytest

from dequant_project_b200 import _native


def cache(**kw):
    a = dict(k=1 << 20, v=1 << 21, k_scale=1 << 22, v_scale=1 << 23, k_open=1 << 24, v_open=1 << 25, n_pages=4,
             n_kv_heads=2, page_size=32, head_dim=128, block=16, n_open=3, page_stride=8192, head_stride=4096,
             row_stride=128, scale_page_stride=4, scale_head_stride=2, open_stride=4096, open_head_stride=2048, codes=0,
             dtype=0)
    a.update(kw)
    return _native.QuantizedKV(*a.values())


CACHES = [
    (dict(k=None), 1, "k must not be null"),
    (dict(v=(1 << 21) + 8), 1, "v must be 16-byte aligned"),
    (dict(k_scale=(1 << 22) + 2), 1, "k_scale must be 4-byte aligned"),
    (dict(v_open=None), 1, "v_open must not be null"),
    (dict(codes=2), 1, "codes must be"),
    (dict(dtype=2), 1, "dtype must be"),
    (dict(head_dim=96), 2, "head_dim 64 and 128, got 96"),
    (dict(page_size=48), 2, "page_size must be 16"),
    (dict(page_size=512), 2, "page_size must be 16"),
    (dict(block=8), 2, "block must be 16, 32 or 64"),
    (dict(block=64), 2, "block must be 16, 32 or 64 and at most a page"),
    (dict(n_kv_heads=0), 1, "n_kv_heads must be in"),
    (dict(n_pages=0), 1, "n_pages must be in"),
    (dict(n_open=0), 1, "n_open must be in"),
    (dict(page_stride=8200), 1, "page stride must be a multiple of 16"),
    (dict(head_stride=0), 1, "head stride must be a multiple of 16"),
    (dict(row_stride=64), 1, "row stride must be a multiple of 16 and at least 128"),
    (dict(scale_page_stride=1), 1, "scales' page stride"),
    (dict(scale_head_stride=1), 1, "scales' head stride"),
    (dict(open_stride=2052), 1, "open blocks' stride"),
    (dict(open_head_stride=1024), 1, "open blocks' head stride"),
]


def rejected(rc, code, msg):
    assert rc == code
    assert msg in _native.lib().dqg_last_error().decode()


def append(kv=None, **kw):
    a = dict(qkv=16, T=3, stride=1024, hq=4, cos=16, sin=16, n=8, rot=128, inter=0, pos=16, qn=None, kn=None, eps=1e-5)
    b = dict(table=16, width=3, tstride=3, open=16, starts=16, lens=16, seqs=2, q_out=16)
    for k, v in kw.items():
        (a if k in a else b)[k] = v
    return _native.lib().dqg_rope_quantized_append(*a.values(), cache() if kv is None else kv, *b.values(), None)


def expand(kv=None, **kw):
    a = dict(table=16, width=3, tstride=3, open=16, lens=16, seqs=2, pages=6, k_out=16, v_out=16, table_out=16)
    a.update(kw)
    return _native.lib().dqg_expand_pages(cache() if kv is None else kv, *a.values(), None)


def decode(kv=None, **kw):
    a = dict(q=16, qs=512, qh=128, seqs=2, hq=4)
    b = dict(table=16, width=3, tstride=3, open=16, lens=16, scale=0.1, out=16, ws=16, bytes=1 << 40)
    for k, v in kw.items():
        (a if k in a else b)[k] = v
    return _native.lib().dqg_quantized_attention(*a.values(), cache() if kv is None else kv, *b.values(), None)


def prompt(kv=None, **kw):
    a = dict(q=16, qs=512, qh=128, T=5, hq=4)
    b = dict(table=16, width=3, tstride=3, open=16, starts=16, lens=16, seqs=2, pages=6, causal=1, scale=0.1, out=16, ws=256,
             bytes=1 << 40)
    for k, v in kw.items():
        (a if k in a else b)[k] = v
    return _native.lib().dqg_quantized_prompt_attention(*a.values(), cache() if kv is None else kv, *b.values(), None)


def sample(params=None, **kw):
    a = dict(logits=16, dtype=0, rows=2, vocab=100, stride=100, uniform=16)
    b = dict(tokens=16, logprobs=16)
    for k, v in kw.items():
        (a if k in a else b)[k] = v
    p = _native.Sampling(**{**dict(temperature=1.0, top_p=1.0), **(params or {})})
    return _native.lib().dqg_sample_tokens(*a.values(), p, *b.values(), None)


@pytest.mark.parametrize("call", [append, expand, decode, prompt], ids=lambda f: f.__name__)
@pytest.mark.parametrize("kw,code,msg", CACHES, ids=lambda v: str(v))
def test_caches(call, kw, code, msg):
    rejected(call(cache(**kw)), code, msg)


SEQS = [
    (dict(seqs=-1), "n_seqs=-1 out of range"),
    (dict(table=None), "block_table must not be null"),
    (dict(width=0), "at least one page"),
    (dict(tstride=2), "at least one page"),
    (dict(open=None), "open_slots must not be null"),
    (dict(lens=6), "kv_lens must be 4-byte aligned"),
]


@pytest.mark.parametrize("call", [append, expand, decode, prompt], ids=lambda f: f.__name__)
@pytest.mark.parametrize("kw,msg", SEQS, ids=lambda v: str(v))
def test_sequences(call, kw, msg):
    rejected(call(**kw), 1, msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=-1), "T=-1 out of range"),
    (dict(stride=1000), "row stride"),
    (dict(stride=1028), "row stride"),
    (dict(hq=3), "must give 1..128 query heads"),
    (dict(rot=7), "rotary_dim must be even"),
    (dict(rot=130), "rotary_dim must be even"),
    (dict(n=0), "at least one position"),
    (dict(qn=16), "given together"),
    (dict(eps=float("nan")), "eps must be non-negative"),
    (dict(qkv=8), "qkv must be 16-byte aligned"),
    (dict(pos=12), "positions must be 8-byte aligned"),
    (dict(starts=None), "q_starts must not be null"),
    (dict(q_out=None), "q_out must not be null"),
    (dict(qn=16, kn=8), "k_norm must be 16-byte aligned"),
], ids=lambda v: str(v))
def test_append(kw, msg):
    rejected(append(**kw), 1, msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(q=24), "q must be 16-byte aligned"),
    (dict(qh=64), "q's strides"),
    (dict(hq=5), "must give 1..128 query heads"),
    (dict(hq=512), "must give 1..128 query heads"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
    (dict(out=8), "out must be 16-byte aligned"),
], ids=lambda v: str(v))
def test_attention(kw, msg):
    rejected(decode(**kw), 1, msg)
    rejected(prompt(**kw), 1, msg)


def test_prompt():
    rejected(prompt(T=-1), 1, "T=-1 out of range")
    rejected(prompt(pages=-1), 1, "n_pages=-1 out of range")
    rejected(prompt(starts=None), 1, "q_starts must not be null")


@pytest.mark.parametrize("kw,code,msg", [
    (dict(pages=-1), 1, "n_pages=-1 out of range"),
    (dict(k_out=8), 1, "k_out must be 16-byte aligned"),
    (dict(v_out=None), 1, "v_out must not be null"),
    (dict(table_out=2), 1, "table_out must be 4-byte aligned"),
], ids=lambda v: str(v))
def test_expand(kw, code, msg):
    rejected(expand(**kw), code, msg)


@pytest.mark.parametrize("kw,params,code,msg", [
    (dict(dtype=3), {}, 1, "dtype must be"),
    (dict(rows=-1), {}, 1, "rows=-1 out of range"),
    (dict(vocab=0), {}, 2, "vocab must be in"),
    (dict(vocab=2 ** 18 + 1), {}, 2, "vocab must be in"),
    (dict(stride=99), {}, 1, "row stride must be at least 100"),
    (dict(logits=None), {}, 1, "logits must not be null"),
    (dict(dtype=2, logits=18), {}, 1, "logits must be 4-byte aligned"),
    (dict(uniform=18), {}, 1, "uniform must be 4-byte aligned"),
    (dict(tokens=20), {}, 1, "tokens must be 8-byte aligned"),
    (dict(logprobs=None), {}, 1, "logprobs must not be null"),
    ({}, dict(temperatures=6), 1, "temperatures must be 4-byte aligned"),
    ({}, dict(top_ks=6), 1, "top_ks must be 4-byte aligned"),
    ({}, dict(top_ps=6), 1, "top_ps must be 4-byte aligned"),
    ({}, dict(min_ps=6), 1, "min_ps must be 4-byte aligned"),
], ids=lambda v: str(v))
def test_sample(kw, params, code, msg):
    rejected(sample(params, **kw), code, msg)


def test_empty_calls_launch_nothing():
    assert append(T=0) == 0 and expand(seqs=0) == 0 and decode(seqs=0) == 0 and prompt(T=0) == 0 and sample(rows=0) == 0
    rejected(_native.lib().dqg_sample_tokens(16, 0, 1, 1, 1, 16, None, 16, 16, None), 1, "params must not be null")


def test_workspace_queries():
    lib, n = _native.lib(), ctypes.c_uint64(0)
    rejected(lib.dqg_quantized_attention_workspace(2, 4, 2, 96, ctypes.byref(n)), 2, "head_dim 64 and 128")
    rejected(lib.dqg_quantized_attention_workspace(2, 4, 3, 128, ctypes.byref(n)), 1, "query heads per KV head")
    rejected(lib.dqg_quantized_attention_workspace(2, 4, 2, 128, None), 1, "bytes must not be null")
    rejected(lib.dqg_quantized_prompt_workspace(cache(block=8), 2, 3, 6, ctypes.byref(n)), 2, "block must be 16")
    rejected(lib.dqg_quantized_prompt_workspace(cache(), 2, 0, 6, ctypes.byref(n)), 1, "table_width=0")
    rejected(lib.dqg_quantized_prompt_workspace(cache(), 2, 3, -1, ctypes.byref(n)), 1, "n_pages=-1")


def test_struct_layouts():
    """As ctypes lays them out: six pointers, thirteen 64-bit counts and two
    32-bit types; four pointers and four 32-bit values."""
    assert ctypes.sizeof(_native.QuantizedKV) == 6 * 8 + 13 * 8 + 2 * 4
    assert ctypes.sizeof(_native.Sampling) == 4 * 8 + 4 * 4
