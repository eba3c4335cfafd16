"""What is measured of the paged-cache operators: a prompt's and a decode
step's path through a KV cache that is held in pages.

Four operators: ``rope_paged_append`` (per-head norms of queries and keys,
position rotation, keys and values into their pages), ``prompt_attention``
(packed prompts or chunks of them over the pages), ``paged_attention`` (one
query token per sequence) and ``shared_prefix_attention`` (the same for a batch
whose sequences begin with the same cached prefix). ``run`` computes each in
plain fp32 torch operations where ``own`` is false, and through
``dequant_project_b200.paged_ops`` where it is true.

Head layouts are those of the decoder's two architectures (32 query and 32
key/value heads; 64 and 8) and of their tensor-parallel shards, plus heads of
64 values. Pages hold [page, kv head, position in page, value]; a sequence's
pages are scattered over the pool in random order, and what lies in a page
behind a sequence's end is stale data of another request.
"""

import math
import random

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases
def _text(values):
    return ",".join(str(v) for v in values)


def _numbers(text):
    return [int(v) for v in text.split(",")]


def _ragged(n, lo, hi, seed):
    """n lengths spread over their logarithm."""
    rng = random.Random(seed)
    return [int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) for _ in range(n)]


def listed():
    return [
        # One decode step of eight sequences: eight tokens rotated and stored.
        {"name": "append step 8", "op": "append", "tokens": 8, "hq": 32, "hkv": 32, "d": 128, "rot": 128,
         "interleaved": False, "norm": False, "page": 16, "skip": 0, "type": "fp16"},
        # A long prompt of the grouped-head architecture, with norms of queries and keys.
        {"name": "append prompt 8192 qk-norm", "op": "append", "tokens": 8192, "hq": 64, "hkv": 8, "d": 128,
         "rot": 128, "interleaved": False, "norm": True, "page": 64, "skip": 0, "type": "bf16"},
        # A packed batch of odd size: interleaved pairs over half of a small head, every 11th token padding.
        {"name": "append 1777 interleaved", "op": "append", "tokens": 1777, "hq": 32, "hkv": 8, "d": 64, "rot": 32,
         "interleaved": True, "norm": False, "page": 16, "skip": 11, "type": "fp16"},
        # One prompt as long as the benchmark's cache.
        {"name": "prompt 2048", "op": "prompt", "q_lens": "2048", "kv_lens": "2048", "hq": 32, "hkv": 32, "d": 128,
         "page": 64, "type": "fp16"},
        # One long prompt with grouped heads: the largest case.
        {"name": "prompt 8192 grouped", "op": "prompt", "q_lens": "8192", "kv_lens": "8192", "hq": 64, "hkv": 8,
         "d": 128, "page": 128, "type": "bf16"},
        # Requests of very different lengths packed into one call, an empty one and a single token among them.
        {"name": "prompt packed ragged", "op": "prompt", "q_lens": "1,37,0,1291,200,2777,64,511,129,5,803,1024,16",
         "kv_lens": "1,37,0,1291,712,2777,64,511,129,5,2003,1024,1040", "hq": 32, "hkv": 8, "d": 64, "page": 16,
         "type": "fp16"},
        # A chunk of a long document whose beginning is cached: few rows, a long axis.
        {"name": "prompt chunk 300 of 30000", "op": "prompt", "q_lens": "300", "kv_lens": "30000", "hq": 64, "hkv": 8,
         "d": 128, "page": 32, "type": "bf16"},
        # The benchmark's decode step: one sequence, 2048 cached positions and the new one.
        {"name": "decode 1 x 2049", "op": "decode", "kv_lens": "2049", "hq": 32, "hkv": 32, "d": 128, "page": 16,
         "type": "fp16"},
        # A serving batch of sixty-four sequences of very different lengths, two of its slots empty.
        {"name": "decode 64 ragged grouped", "op": "decode", "kv_lens": _text([0, 1, 0] + _ragged(61, 900, 16000, 1)),
         "hq": 64, "hkv": 8, "d": 128, "page": 16, "type": "bf16"},
        # One rank's heads at tensor-parallel width 8.
        {"name": "decode 8 shard", "op": "decode", "kv_lens": _text([4097, 4001, 3000, 4097, 2500, 4090, 128, 3333]),
         "hq": 8, "hkv": 1, "d": 128, "page": 32, "type": "fp16"},
        # Sixteen conversations behind one system prompt, multi-head.
        {"name": "shared prefix 16 x 2000", "op": "shared", "prefix": 2000,
         "kv_lens": _text([0] + _ragged(15, 8, 600, 2)), "hq": 32, "hkv": 32, "d": 128, "page": 16, "type": "fp16"},
        # Many samples of one long document, grouped heads.
        {"name": "shared prefix 128 x 16384 grouped", "op": "shared", "prefix": 16384,
         "kv_lens": _text(_ragged(128, 16, 1100, 3)), "hq": 64, "hkv": 8, "d": 128, "page": 64, "type": "bf16"},
    ]


def _pairs(case):
    """Query-key pairs per query head that a prompt case's rows see."""
    total = 0
    for ql, kl in zip(_numbers(case["q_lens"]), _numbers(case["kv_lens"])):
        first = kl - ql + 1  # keys that the first query sees
        total += sum(max(0, first + i) for i in range(ql))
    return total


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    hq, hkv, d = rng.choice([(32, 32, 128), (64, 8, 128), (8, 1, 128), (16, 16, 128), (28, 4, 128), (32, 8, 64),
                             (16, 2, 64), (6, 2, 128)])
    case = {"hq": hq, "hkv": hkv, "d": d, "page": rng.choice([16, 32, 64, 128]), "type": rng.choice(["fp16", "bf16"])}
    op = rng.choice(["append", "prompt", "decode", "shared"])
    if op == "append":
        rot = rng.choice([d, d, d // 2, d // 4])
        case.update(op=op, tokens=spread(1, 8192), rot=rot, interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.5, skip=rng.choice([0, 0, 7, 13]))
        return case
    if op == "prompt":
        n = spread(1, 16)
        ql = [spread(1, 6000 // n) if rng.random() < 0.93 else 0 for _ in range(n)]
        ql[0] = max(ql[0], 1)
        kl = [q + (spread(1, 12000000 // max(sum(ql), 800)) if rng.random() < 0.4 else 0) for q in ql]
        case.update(op=op, q_lens=_text(ql), kv_lens=_text(kl))
        return case
    n = spread(1, 96)
    longest = 16000 if n * hkv <= 512 else 4000
    kl = [spread(1, longest) if rng.random() < 0.95 else 0 for _ in range(n)]
    if op == "decode":
        kl[0] = max(kl[0], 1)
        case.update(op=op, kv_lens=_text(kl))
        return case
    n = spread(2, 128)
    case.update(op=op, prefix=spread(100, 16000 if n * hkv <= 1024 else 3000), kv_lens=_text([spread(1, 900) if rng.random() < 0.95 else 0
                                                                 for _ in range(n)]))
    return case


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    row = hkv * d * 2 * 2  # a position's key and value rows, 16-bit
    if case["op"] == "append":
        t = case["tokens"]
        kept = t - (len(range(0, t, case["skip"])) if case["skip"] else 0)
        read = t * (hq + 2 * hkv) * d * 2 + t * 16 + min(t, 8192) * case["rot"] * 4
        return {"bytes": read + t * hq * d * 2 + kept * row, "flops": 3 * t * (hq + hkv) * case["rot"]}
    if case["op"] == "prompt":
        t, kv = sum(_numbers(case["q_lens"])), sum(_numbers(case["kv_lens"]))
        return {"bytes": 2 * t * hq * d * 2 + kv * row, "flops": 4 * d * hq * _pairs(case)}
    lens = _numbers(case["kv_lens"])
    n, kv, p = len(lens), sum(lens), case.get("prefix", 0)
    return {"bytes": 2 * n * hq * d * 2 + (kv + p) * row, "flops": 4 * d * hq * (kv + n * p)}


# ---------------------------------------------------------------- the inputs
def _pool(gen, lens, hkv, d, page, dtype):
    """Key and value pools, and the table of scattered pages that the lengths
    take; the pool has a few pages more than they need."""
    counts = [-(-n // page) for n in lens]
    n_pages = sum(counts) + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), max(1, max(counts))), dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    k = torch.randn((n_pages, hkv, page, d), generator=gen, device="cuda").to(dtype)
    v = torch.randn((n_pages, hkv, page, d), generator=gen, device="cuda").to(dtype)
    return k, v, table


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    hq, hkv, d, page, dtype = case["hq"], case["hkv"], case["d"], case["page"], _TYPES[case["type"]]
    state = {"op": case["op"], "hq": hq}
    if case["op"] == "append":
        t, rot = case["tokens"], case["rot"]
        k, v, table = _pool(gen, [t], hkv, d, page, dtype)
        at = torch.arange(t, device="cuda")
        slots = table[0].long()[at // page] * page + at % page
        if case["skip"]:
            slots[::case["skip"]] = -1
        # A few requests' tokens in a row, each counting from a place of its own.
        length = -(-t // 3)
        start = torch.randint(0, 8192 - min(length, 8191), (3,), generator=gen, device="cuda")
        angle = torch.arange(8192, dtype=torch.float64, device="cuda")[:, None] * (
            10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot))
        state.update(qkv=torch.randn((t, (hq + 2 * hkv) * d), generator=gen, device="cuda").to(dtype),
                     cos=angle.cos().float(), sin=angle.sin().float(),
                     positions=start[at // length] + at % length, slots=slots, k_pages=k, v_pages=v,
                     interleaved=case["interleaved"], eps=1e-5, q_norm=None, k_norm=None)
        if case["norm"]:
            w = 1.0 + 0.1 * torch.randn((2, d), generator=gen, device="cuda")
            state.update(q_norm=w[0].to(dtype), k_norm=w[1].to(dtype))
        return state
    lens = _numbers(case["kv_lens"])
    k, v, table = _pool(gen, lens + [case.get("prefix", 0)], hkv, d, page, dtype)
    width = max(1, max(-(-n // page) for n in lens))
    rows = sum(_numbers(case["q_lens"])) if case["op"] == "prompt" else len(lens)
    state.update(q=torch.randn((rows, hq, d), generator=gen, device="cuda").to(dtype), k_pages=k, v_pages=v,
                 block_table=table[:-1, :width].contiguous(),
                 kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), longest=max(lens))
    if case["op"] == "prompt":
        ql = _numbers(case["q_lens"])
        starts = [0]
        for n in ql:
            starts.append(starts[-1] + n)
        state.update(q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), longest_q=max(ql))
    if case["op"] == "shared":
        state.update(prefix=case["prefix"], prefix_table=table[-1, :-(-case["prefix"] // page)].contiguous())
    return state


# ------------------------------------------------------------ the plain forms
def _rows_of(pages, table, longest):
    """fp32 [n, kv heads, longest, d]: the cached rows that a table's pages hold."""
    n, (_, hkv, page, d) = table.shape[0], pages.shape
    got = pages[table[:, :max(1, -(-longest // page))].long()].float()
    return got.transpose(1, 2).reshape(n, hkv, -1, d)[:, :, :longest]


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v over the keys that `seen` marks, and zero in
    rows that see none. q [n, kv heads, rows, d], seen [n, 1, rows, keys]."""
    s = (q @ k.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    s = torch.where(seen, s, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    return (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    part, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    c, s = cos[:, None], sin[:, None]
    lo, hi = a * c - b * s, b * c + a * s
    part = torch.stack([lo, hi], -1).flatten(-2) if interleaved else torch.cat([lo, hi], -1)
    return torch.cat([part, rest], -1)


def _plain_append(s):
    k_pages, v_pages, hq = s["k_pages"], s["v_pages"], s["hq"]
    _, hkv, page, d = k_pages.shape
    t = s["qkv"].shape[0]
    x = s["qkv"].float().view(t, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if s["q_norm"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + s["eps"]) * s["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + s["eps"]) * s["k_norm"].float()
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q, k = _rotate(q, cos, sin, s["interleaved"]), _rotate(k, cos, sin, s["interleaved"])
    # Tokens without a slot write what the first token that has one writes, once more.
    kept = s["slots"] >= 0
    row = torch.where(kept, torch.arange(t, device=kept.device), kept.int().argmax())
    slot = s["slots"][row].clamp(min=0)
    live = kept.any()
    at = (slot // page, slice(None), slot % page)
    k_pages[at] = torch.where(live, k[row].to(k_pages.dtype), k_pages[at])
    v_pages[at] = torch.where(live, v[row].to(v_pages.dtype), v_pages[at])
    return q.to(s["qkv"].dtype), k_pages, v_pages


def _plain_prompt(s):
    q, starts, lens = s["q"], s["q_starts"].long(), s["kv_lens"].long()
    t, hq, d = q.shape
    hkv, n, lq, lk = s["k_pages"].shape[1], lens.shape[0], max(1, s["longest_q"]), max(1, s["longest"])
    i, j = torch.arange(lq, device=q.device), torch.arange(lk, device=q.device)
    counts = starts[1:] - starts[:-1]
    rows = (starts[:-1, None] + i).clamp(max=t - 1)
    qp = q[rows].float().view(n, lq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    k, v = _rows_of(s["k_pages"], s["block_table"], lk), _rows_of(s["v_pages"], s["block_table"], lk)
    v = torch.where((j < lens[:, None])[:, None, :, None], v, 0.0)
    ends = (lens - counts)[:, None] + i + 1
    seen = (j < ends[:, :, None]) & (j < lens[:, None, None])
    o = _attend(qp, k, v, seen[:, None].repeat(1, 1, hq // hkv, 1))
    o = o.view(n, hkv, hq // hkv, lq, d).permute(0, 3, 1, 2, 4).reshape(n, lq, hq, d)
    token = torch.arange(t, device=q.device)
    which = torch.searchsorted(starts[1:].contiguous(), token, right=True)
    return o[which, token - starts[which]].to(q.dtype)


def _plain_decode(s):
    q, lens, longest = s["q"], s["kv_lens"].long(), max(1, s["longest"])
    n, hq, d = q.shape
    hkv = s["k_pages"].shape[1]
    k, v = _rows_of(s["k_pages"], s["block_table"], longest), _rows_of(s["v_pages"], s["block_table"], longest)
    seen = torch.arange(longest, device=q.device) < lens[:, None]
    qh = q.float().view(n, hkv, hq // hkv, d)
    if s["op"] == "shared":
        one = s["prefix_table"][None]
        pk, pv = _rows_of(s["k_pages"], one, s["prefix"]), _rows_of(s["v_pages"], one, s["prefix"])
        k = torch.cat([pk.expand(n, -1, -1, -1), k], 2)
        v = torch.cat([pv.expand(n, -1, -1, -1), v], 2)
        seen = torch.cat([seen.new_ones((n, s["prefix"])), seen], 1)
    o = _attend(qh, k, torch.where(seen[:, None, :, None], v, 0.0), seen[:, None, None])
    return o.reshape(n, hq, d).to(q.dtype)


def run(state):
    s = state
    if not own:
        return {"append": _plain_append, "prompt": _plain_prompt, "decode": _plain_decode,
                "shared": _plain_decode}[s["op"]](s)
    from dequant_project_b200 import paged_ops
    if s["op"] == "append":
        q = paged_ops.rope_paged_append(s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_pages"],
                                        s["v_pages"], s["hq"], interleaved=s["interleaved"], q_norm=s["q_norm"],
                                        k_norm=s["k_norm"], eps=s["eps"])
        return q, s["k_pages"], s["v_pages"]
    if s["op"] == "prompt":
        return paged_ops.prompt_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["q_starts"],
                                          s["kv_lens"])
    if s["op"] == "decode":
        return paged_ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["kv_lens"])
    return paged_ops.shared_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["prefix_table"], s["prefix"],
                                             s["block_table"], s["kv_lens"])


# ---------------------------------------------------------- the definitions
def _exact_append(case, s):
    hq, hkv, d, page, rot = case["hq"], case["hkv"], case["d"], case["page"], case["rot"]
    x = s["qkv"].double().view(case["tokens"], hq + 2 * hkv, d)
    heads = x[:, :hq + hkv].clone()
    if case["norm"]:
        mean = (heads ** 2).sum(-1, keepdim=True) / d
        weight = torch.cat([s["q_norm"].double().expand(hq, d), s["k_norm"].double().expand(hkv, d)])
        heads = heads / torch.sqrt(mean + s["eps"]) * weight
    turned, i = heads.clone(), torch.arange(rot // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
    # The angles' cosines and sines are those that the call is given.
    c, n = (s[name].double()[s["positions"]][:, None] for name in ("cos", "sin"))
    turned[..., a] = c * heads[..., a] - n * heads[..., b]
    turned[..., b] = n * heads[..., a] + c * heads[..., b]
    k, v = s["k_pages"].double(), s["v_pages"].double()
    token = torch.nonzero(s["slots"] >= 0)[:, 0]
    slot = s["slots"][token]
    k[slot // page, :, slot % page] = turned[token, hq:]
    v[slot // page, :, slot % page] = x[token, hq + hkv:]
    return turned[:, :hq], k, v


def _exact_rows(q, k, v, ends):
    """One KV head in 64 bits: q [rows, d], and row r sees the first ends[r] of the keys."""
    score = torch.einsum("rd,td->rt", q, k) * (q.shape[1] ** -0.5)
    hidden = torch.arange(k.shape[0], device=q.device)[None] >= ends[:, None]
    p = torch.softmax(score.masked_fill(hidden, float("-inf")), 1)
    return torch.einsum("rt,td->rd", p.masked_fill(hidden, 0.0).nan_to_num(0.0), v)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens, g, at = _numbers(case["kv_lens"]), hq // hkv, 0
    counts = _numbers(case["q_lens"]) if case["op"] == "prompt" else [1] * len(lens)
    for b, (n, c) in enumerate(zip(lens, counts)):
        pages = s["block_table"][b, :-(-n // page)].long()
        keep = [torch.arange(n, device="cuda")]
        if case["op"] == "shared":
            pages = torch.cat([s["prefix_table"].long(), pages])
            p = case["prefix"]
            keep = [torch.arange(p, device="cuda"), -(-p // page) * page + keep[0]]
            n += p
        if n and c:
            ends = torch.arange(n - c + 1, n + 1, device="cuda").repeat_interleave(g)
            keep = torch.cat(keep)
            for h in range(hkv):
                k, v = (s[name][pages, h].reshape(-1, d)[keep].double() for name in ("k_pages", "v_pages"))
                q = s["q"][at:at + c, h * g:(h + 1) * g].double().reshape(-1, d)
                # Heads of one sequence share their mask: a few thousand rows at a time.
                for r in range(0, c * g, 8192):
                    part = _exact_rows(q[r:r + 8192], k, v, ends[r:r + 8192])
                    idx = torch.arange(r, min(r + 8192, c * g), device="cuda")
                    out[at + idx // g, h * g + idx % g] = part
        at += c
    return out
