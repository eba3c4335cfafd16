"""What is measured of the serving path over a key/value cache held in 8 bits,
and of the draw of the tokens that ends each of its steps.

Four operators, each in plain fp32 (sums of a draw: fp64) torch operations
where ``own`` is false and through ``dequant_project_b200`` where it is true:

* ``rope_quantized_append``: per-head norms and rotation, and keys and values
  into 8-bit pages (int8 or e4m3 codes with an fp32 scale for every block of
  positions and head; the rows of a block that is not complete wait in 16
  bits). What it has stored is read back with ``expanded_pages``, as 16-bit
  pages.
* ``quantized_attention``: one query token per sequence over such a cache.
* ``quantized_prompt_attention``: packed prompts, or chunks of them, over it.
* ``sample_tokens``: the next token of each row of logits, with temperature,
  top-k, top-p and min-p, from one given random number a row.

Head layouts are those of the decoder's two architectures (32 query and 32
key/value heads; 64 and 8) and of their tensor-parallel shards, plus heads of
64 values; vocabularies those of the two architectures. A sequence's pages are
scattered over the pool, what lies in a page behind its complete blocks is
stale data of another request, and blocks differ in their largest value as
keys and values of different tokens do.
"""

import math
import random

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
_LEAST = 2.0 ** -126  # of a scale


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
        # One decode step of eight sequences: eight tokens, two of which complete their block.
        {"name": "store step 8", "op": "store", "q_lens": "1,1,1,1,1,1,1,1", "kv_lens": "1,352,17,2049,300,64,777,1031",
         "pad": 0, "hq": 32, "hkv": 32, "d": 128, "rot": 128, "interleaved": False, "norm": False, "page": 16,
         "block": 16, "codes": "int8", "type": "fp16"},
        # A long prompt of the grouped-head architecture, with norms of queries and keys.
        {"name": "store prompt 8192 qk-norm", "op": "store", "q_lens": "8192", "kv_lens": "8192", "pad": 0, "hq": 64,
         "hkv": 8, "d": 128, "rot": 128, "interleaved": False, "norm": True, "page": 64, "block": 32, "codes": "e4m3",
         "type": "bf16"},
        # Chunks of several prompts that begin and end inside blocks; interleaved pairs over half of a small head,
        # and rows of padding behind the last sequence.
        {"name": "store ragged chunks", "op": "store", "q_lens": "500,0,3,777,1,280,129,64",
         "kv_lens": "1003,40,18,777,16,300,2000,64", "pad": 46, "hq": 32, "hkv": 8, "d": 64, "rot": 32,
         "interleaved": True, "norm": False, "page": 32, "block": 16, "codes": "int8", "type": "fp16"},
        # The benchmark's decode step: one sequence, 2048 cached positions and the new one.
        {"name": "decode 1 x 2049", "op": "decode", "kv_lens": "2049", "hq": 32, "hkv": 32, "d": 128, "page": 16,
         "block": 16, "codes": "int8", "type": "fp16"},
        # A serving batch of sixty-four sequences of very different lengths, two of its slots empty: the largest decode.
        {"name": "decode 64 ragged grouped", "op": "decode", "kv_lens": _text([0, 1, 0] + _ragged(61, 900, 16000, 1)),
         "hq": 64, "hkv": 8, "d": 128, "page": 64, "block": 16, "codes": "int8", "type": "bf16"},
        # One rank's heads at tensor-parallel width 8, with the other 8-bit type and the widest blocks.
        {"name": "decode 8 shard", "op": "decode", "kv_lens": "4097,4001,2999,4096,2500,4090,128,3333", "hq": 8, "hkv": 1,
         "d": 128, "page": 128, "block": 64, "codes": "e4m3", "type": "fp16"},
        # One prompt as long as the benchmark's cache.
        {"name": "prompt 2048", "op": "prompt", "q_lens": "2048", "kv_lens": "2048", "hq": 32, "hkv": 32, "d": 128,
         "page": 64, "block": 16, "codes": "int8", "type": "fp16"},
        # A chunk of a long document whose beginning is cached: few rows, a long axis.
        {"name": "prompt chunk 300 of 30000", "op": "prompt", "q_lens": "300", "kv_lens": "30000", "hq": 64, "hkv": 8,
         "d": 128, "page": 32, "block": 32, "codes": "int8", "type": "bf16"},
        # Requests of very different lengths packed into one call, an empty one and a single token among them.
        {"name": "prompt packed ragged", "op": "prompt", "q_lens": "1,37,0,1291,200,2777,64,511,129,5,803,1024,16",
         "kv_lens": "1,37,0,1291,712,2777,64,511,129,5,2003,1024,1040", "hq": 32, "hkv": 8, "d": 64, "page": 16,
         "block": 16, "codes": "e4m3", "type": "fp16"},
        # The next token of one conversation, every filter on.
        {"name": "sample 1 x 32000", "op": "sample", "rows": 1, "vocab": 32000, "top_k": True, "top_p": True,
         "min_p": False, "greedy": False, "type": "fp16"},
        # A serving batch whose requests ask for different things, greedy ones among them.
        {"name": "sample 64 x 128256 mixed", "op": "sample", "rows": 64, "vocab": 128256, "top_k": True, "top_p": True,
         "min_p": True, "greedy": True, "type": "fp16"},
        # Many samples of fp32 logits from the whole distribution.
        {"name": "sample 256 x 32000 fp32", "op": "sample", "rows": 256, "vocab": 32000, "top_k": False, "top_p": False,
         "min_p": False, "greedy": False, "type": "fp32"},
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

    op = rng.choice(["store", "decode", "prompt", "sample"])
    if op == "sample":
        vocab = spread(1000, 130000)
        return {"op": op, "rows": spread(1, min(256, 8200000 // vocab)), "vocab": vocab, "top_k": rng.random() < 0.5,
                "top_p": rng.random() < 0.6, "min_p": rng.random() < 0.3, "greedy": rng.random() < 0.3,
                "type": rng.choice(["fp16", "bf16", "fp32"])}
    hq, hkv, d = rng.choice([(32, 32, 128), (64, 8, 128), (8, 1, 128), (16, 16, 128), (28, 4, 128), (32, 8, 64),
                             (16, 2, 64), (6, 2, 128), (24, 2, 64)])
    block = rng.choice([16, 16, 32, 64])
    case = {"hq": hq, "hkv": hkv, "d": d, "page": max(block, rng.choice([16, 32, 64, 128])), "block": block,
            "codes": rng.choice(["int8", "e4m3"]), "type": rng.choice(["fp16", "bf16"])}
    if op == "decode":
        n = spread(1, 96)
        longest = 16000 if n * hkv <= 512 else 4000
        kl = [spread(1, longest) if rng.random() < 0.95 else 0 for _ in range(n)]
        kl[0] = max(kl[0], 1)
        case.update(op=op, kv_lens=_text(kl))
        return case
    n = spread(1, 16)
    if op == "store":
        steps = rng.random() < 0.3
        ql = [1 if steps else (spread(1, 6000 // n) if rng.random() < 0.93 else 0) for _ in range(n)]
        ql[0] = max(ql[0], 1)
        kl = [q + (spread(1, 3000) if rng.random() < 0.6 else 0) for q in ql]
        case.update(op=op, q_lens=_text(ql), kv_lens=_text(kl), pad=rng.choice([0, 0, 5, 40]),
                    rot=rng.choice([d, d, d // 2, d // 4]), interleaved=rng.random() < 0.4, norm=rng.random() < 0.5)
        return case
    ql = [spread(1, 4000 // n) if rng.random() < 0.93 else 0 for _ in range(n)]
    ql[0] = max(ql[0], 1)
    kl = [q + (spread(1, 8000000 // max(sum(ql), 800)) if rng.random() < 0.4 else 0) for q in ql]
    case.update(op=op, q_lens=_text(ql), kv_lens=_text(kl))
    return case


def _tail(case, q, n):
    """First position of the page in which a stored chunk's oldest open or new row lies."""
    first = max(0, n - max(q, 1)) // case["block"] * case["block"]
    return first // case["page"] * case["page"]


def work(case):
    if case["op"] == "sample":
        rows, size = case["rows"], torch.finfo(_TYPES[case["type"]]).bits // 8
        flags = 4 * (1 + case["top_k"] + case["top_p"] + case["min_p"])
        return {"bytes": rows * (case["vocab"] * size + flags + 4 + 12), "flops": 3 * rows * case["vocab"]}
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    lens = _numbers(case["kv_lens"])
    open_rows = sum(n % block for n in lens)
    blocks = sum(n // block for n in lens)
    pages = blocks * hkv * (block * d + 4) * 2 + open_rows * hkv * d * 2 * 2
    if case["op"] == "store":
        ql, page = _numbers(case["q_lens"]), case["page"]
        t = sum(ql) + case["pad"]
        done = sum(n // block - (n - q) // block for q, n in zip(ql, lens))
        old = sum((n - q) % block for q, n in zip(ql, lens) if q and (n - q) // block < n // block)
        new = sum(min(q, n % block) for q, n in zip(ql, lens))
        tails = [n - _tail(case, q, n) for q, n in zip(ql, lens)]
        back = sum(-(-n // page) * page for n in tails)
        read = t * (hq + 2 * hkv) * d * 2 + t * 8 + t * case["rot"] * 4 + old * hkv * d * 4
        back_read = sum(n // block for n in tails) * hkv * (block * d + 4) * 2 + open_rows * hkv * d * 4
        return {"bytes": read + t * hq * d * 2 + done * hkv * (block * d + 4) * 2 + new * hkv * d * 4 + back_read +
                back * hkv * d * 4, "flops": 3 * t * (hq + hkv) * case["rot"] + 4 * t * hkv * d}
    if case["op"] == "prompt":
        t = sum(_numbers(case["q_lens"]))
        return {"bytes": 2 * t * hq * d * 2 + pages, "flops": 4 * d * hq * _pairs(case)}
    return {"bytes": 2 * len(lens) * hq * d * 2 + pages, "flops": 4 * d * hq * sum(lens)}


# ---------------------------------------------------------------- the inputs
def _quantized(x, block, codes):
    """Codes and scales of rows [..., rows, d], a scale for every `block` rows."""
    dtype, most = _CODES[codes]
    y = x.float().unflatten(-2, (-1, block))
    scale = (y.abs().amax((-1, -2), keepdim=True) / most).clamp(min=_LEAST)
    c = y / scale
    c = torch.round(c).to(dtype) if codes == "int8" else c.to(dtype)
    return c.flatten(-3, -2), scale[..., 0, 0]


def _cache(gen, case, lens):
    """Pools of 8-bit pages and open blocks, and the table and open slots of
    the sequences; the pools have a few pages and slots more than they take."""
    hkv, d, page, block, dtype = case["hkv"], case["d"], case["page"], case["block"], _TYPES[case["type"]]
    counts = [-(-n // page) for n in lens]
    n_pages, n_slots = sum(counts) + 3, len(lens) + 2
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), max(1, max(counts))), dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    cache = []
    for _ in range(2):
        x = torch.randn((n_pages, hkv, page, d), generator=gen, device="cuda").to(dtype)
        size = torch.exp(0.5 * torch.randn((n_pages, hkv, page, 1), generator=gen, device="cuda")).to(dtype)
        cache.append(_quantized(x * size, block, case["codes"]))
    opened = [torch.randn((n_slots, hkv, block, d), generator=gen, device="cuda").to(dtype) for _ in range(2)]
    slots = torch.randperm(n_slots, generator=gen, device="cuda")[:len(lens)].to(torch.int32)
    (k, ks), (v, vs) = cache
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "k_open": opened[0], "v_open": opened[1], "table": table,
            "slots": slots}


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"op": case["op"]}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]

        def uniform(lo, hi):
            return lo + (hi - lo) * torch.rand(rows, generator=gen, device="cuda")

        logits = 3.0 * torch.randn((rows, vocab), generator=gen, device="cuda")
        # A third of the rows may take a few tokens only, as a grammar's do.
        fenced = torch.rand((rows, vocab), generator=gen, device="cuda") < 0.95
        logits = logits.masked_fill(fenced & (torch.arange(rows, device="cuda") % 3 == 2)[:, None], float("-inf"))
        heat = uniform(0.3, 1.4)
        if case["greedy"]:
            heat = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.25, 0.0, heat)
        k = torch.exp(uniform(0.0, 7.0)).int()
        s.update(logits=logits.to(_TYPES[case["type"]]), uniform=uniform(0.0, 1.0).clamp(max=1 - 2.0 ** -24),
                 temperature=heat, top_k=torch.where(k > 900, 0, k) if case["top_k"] else None,
                 top_p=uniform(0.5, 1.02) if case["top_p"] else None,
                 min_p=uniform(0.0, 0.2) if case["min_p"] else None)
        return s
    hq, hkv, d, page, dtype = case["hq"], case["hkv"], case["d"], case["page"], _TYPES[case["type"]]
    lens = _numbers(case["kv_lens"])
    s.update(_cache(gen, case, lens), hq=hq, block=case["block"], codes=case["codes"], kv_lens=_ints(lens),
             longest=max(lens))
    if case["op"] == "decode":
        s["q"] = torch.randn((len(lens), hq, d), generator=gen, device="cuda").to(dtype)
        return s
    ql = _numbers(case["q_lens"])
    starts = [0]
    for n in ql:
        starts.append(starts[-1] + n)
    s.update(q_starts=_ints(starts), longest_q=max(ql))
    if case["op"] == "prompt":
        s.update(q=torch.randn((starts[-1], hq, d), generator=gen, device="cuda").to(dtype),
                 total_pages=sum(-(-n // page) for n in lens))
        return s
    t, rot = starts[-1] + case["pad"], case["rot"]
    place = [p for q, n in zip(ql, lens) for p in range(n - q, n)] + [0] * case["pad"]
    angle = torch.arange(16384, dtype=torch.float64, device="cuda")[:, None] * (
        10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot))
    s.update(qkv=torch.randn((t, (hq + 2 * hkv) * d), generator=gen, device="cuda").to(dtype), cos=angle.cos().float(),
             sin=angle.sin().float(), positions=torch.tensor(place, dtype=torch.int64, device="cuda"),
             interleaved=case["interleaved"], eps=1e-5, q_norm=None, k_norm=None)
    if case["norm"]:
        w = 1.0 + 0.1 * torch.randn((2, d), generator=gen, device="cuda")
        s.update(q_norm=w[0].to(dtype), k_norm=w[1].to(dtype))
    # What is read back: each sequence's pages from the first that the call touches on.
    first = [_tail(case, q, n) for q, n in zip(ql, lens)]
    tails = [n - f for n, f in zip(lens, first)]
    width = max(1, max(-(-n // page) for n in tails))
    back = torch.zeros((len(lens), width), dtype=torch.int32, device="cuda")
    for i, (f, n) in enumerate(zip(first, tails)):
        c = -(-n // page)
        back[i, :c] = s["table"][i, f // page:f // page + c]
    s.update(back_table=back, back_lens=_ints(tails), back_pages=sum(-(-n // page) for n in tails),
             longest_back=width * page, span=max(-(-(q + case["block"]) // case["block"]) + 1 for q in ql))
    return s


# ------------------------------------------------------------ the plain forms
def _values(codes, scale, block):
    """fp32 values of pages [..., page, d] of codes."""
    return codes.float() * scale.repeat_interleave(block, -1)[..., None]


def _rows_of(s, name, table, lens, longest):
    """fp32 [n, kv heads, longest, d]: a cache's positions, the open rows among
    them, zeros behind each sequence's end."""
    codes, scale, opened, block = s[name], s[name + "_scale"], s[name + "_open"], s["block"]
    hkv, page, d = codes.shape[1:]
    pick = table[:, :max(1, -(-longest // page))].long()
    x = _values(codes.view(torch.uint8)[pick].view(codes.dtype), scale[pick], block)
    x = x.transpose(1, 2).reshape(table.shape[0], hkv, -1, d)[:, :, :longest]
    t = torch.arange(longest, device=x.device)
    lens = lens.long()[:, None]
    done = lens - lens % block
    late = opened[s["slots"].long()[:, None], :, (t - done).clamp(0, block - 1)].float().transpose(1, 2)
    x = torch.where((t < done)[:, None, :, None], x, late)
    return torch.where((t < lens)[:, None, :, None], x, 0.0)


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
    c, n = cos[:, None], sin[:, None]
    lo, hi = a * c - b * n, b * c + a * n
    part = torch.stack([lo, hi], -1).flatten(-2) if interleaved else torch.cat([lo, hi], -1)
    return torch.cat([part, rest], -1)


def _plain_put(s, name, new):
    """New rows [T, kv heads, d] of the 16-bit type into a cache: complete
    blocks in 8 bits, the others' rows into the open blocks."""
    codes, scale, opened, block = s[name], s[name + "_scale"], s[name + "_open"], s["block"]
    starts, lens, table, slots = s["q_starts"].long(), s["kv_lens"].long(), s["table"].long(), s["slots"].long()
    _, hkv, page, d = codes.shape
    begin = lens - (starts[1:] - starts[:-1])
    base = begin - begin % block
    # Every position from the oldest open one on, by sequence and block.
    at = base[:, None] + torch.arange(s["span"] * block, device=new.device)
    row = (starts[:-1, None] + at - begin[:, None]).clamp(0, new.shape[0] - 1)
    x = torch.where((at >= begin[:, None])[..., None, None], new[row],
                    opened[slots[:, None], :, at % block])
    c, f = _quantized(x.view(len(lens), -1, block, hkv, d).transpose(2, 3), block, s["codes"])
    f = f[..., 0]  # [n, blocks, kv heads]
    block_at = at[:, ::block]
    whole = (block_at + block <= lens[:, None]) & (lens > begin)[:, None]
    # Blocks that are not complete write what the first complete one does, once more; without any, what is there.
    n, i = whole.shape[1], torch.arange(whole.numel(), device=new.device)
    pick = torch.where(whole.flatten(), i, whole.flatten().int().argmax())
    b, p = pick // n, block_at.flatten()[pick]
    to = table[b, (p // page).clamp(max=table.shape[1] - 1)]
    part = (p % page) // block
    live = whole.any()
    pool = codes.view(torch.uint8).unflatten(2, (-1, block))  # [pages, kv heads, parts, block, d]
    pool[to, :, part] = torch.where(live, c.view(torch.uint8).flatten(0, 1)[pick], pool[to, :, part])
    scale[to, :, part] = torch.where(live, f.flatten(0, 1)[pick], scale[to, :, part])
    # Open rows: the new ones of blocks that are not complete.
    place = (lens - lens % block)[:, None] + torch.arange(block, device=new.device)
    fresh = (place >= begin[:, None]) & (place < lens[:, None])
    row = (starts[:-1, None] + place - begin[:, None]).clamp(0, new.shape[0] - 1)
    opened[slots] = torch.where(fresh[..., None, None], new[row], opened[slots].transpose(1, 2)).transpose(1, 2)


def _plain_store(s):
    qkv, hq = s["qkv"], s["hq"]
    hkv, page, d = s["k"].shape[1:]
    x = qkv.float().view(qkv.shape[0], hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if s["q_norm"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + s["eps"]) * s["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + s["eps"]) * s["k_norm"].float()
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q, k = _rotate(q, cos, sin, s["interleaved"]), _rotate(k, cos, sin, s["interleaved"])
    _plain_put(s, "k", k.to(qkv.dtype))
    _plain_put(s, "v", v.to(qkv.dtype))
    # Read back as pages, one sequence's after the other's.
    counts = (s["back_lens"].long() + page - 1) // page
    n = s["back_pages"]
    seq = torch.repeat_interleave(torch.arange(len(counts), device=qkv.device), counts, output_size=n)
    part = torch.arange(n, device=qkv.device) - (counts.cumsum(0) - counts)[seq]
    pages = []
    for name in ("k", "v"):
        rows = _rows_of(s, name, s["back_table"], s["back_lens"], s["longest_back"])
        pages.append(rows.unflatten(2, (-1, page)).transpose(1, 2)[seq, part].to(qkv.dtype))
    return q.to(qkv.dtype), *pages, s["k_scale"], s["v_scale"], s["k_open"], s["v_open"]


def _plain_prompt(s):
    q, starts, lens = s["q"], s["q_starts"].long(), s["kv_lens"].long()
    t, hq, d = q.shape
    hkv, n, lq, lk = s["k"].shape[1], lens.shape[0], max(1, s["longest_q"]), max(1, s["longest"])
    i, j = torch.arange(lq, device=q.device), torch.arange(lk, device=q.device)
    counts = starts[1:] - starts[:-1]
    rows = (starts[:-1, None] + i).clamp(max=t - 1)
    qp = q[rows].float().view(n, lq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    k, v = (_rows_of(s, name, s["table"], lens, lk) for name in ("k", "v"))
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
    hkv = s["k"].shape[1]
    k, v = (_rows_of(s, name, s["table"], lens, longest) for name in ("k", "v"))
    seen = torch.arange(longest, device=q.device) < lens[:, None]
    o = _attend(q.float().view(n, hkv, hq // hkv, d), k, v, seen[:, None, None])
    return o.reshape(n, hq, d).to(q.dtype)


def _plain_sample(s):
    x, heat = s["logits"].double(), s["temperature"].double()[:, None]
    vocab = x.shape[1]
    top, order = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(vocab, device=x.device)
    w = torch.where(top.isneginf(), 0.0, torch.exp((top - top[:, :1]) / torch.where(heat > 0, heat, 1.0)))
    kept = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        kept = (rank < k) | (k <= 0)
    if s["top_p"] is not None:
        within = torch.where(kept, w, 0.0)
        before = within.cumsum(1) - within
        p = s["top_p"].double()[:, None]
        kept = kept & ((before < p * within.sum(1, keepdim=True)) | (p >= 1))
    if s["min_p"] is not None:
        kept = kept & (w >= s["min_p"].double()[:, None])
    kept = torch.where(heat > 0, kept, rank == 0)
    # Back in the order of the vocabulary, where the draw is made.
    w = torch.zeros_like(w).scatter(1, order, torch.where(kept, w, 0.0))
    run_sum = w.cumsum(1)
    total = run_sum[:, -1:]
    token = (run_sum <= s["uniform"].double()[:, None] * total).sum(1, keepdim=True)
    last = vocab - 1 - (w.flip(1) > 0).int().argmax(1, keepdim=True)
    token = torch.minimum(token, last)
    return token[:, 0], (w.gather(1, token) / total).log()[:, 0].float()


def run(state):
    s = state
    if not own:
        return {"store": _plain_store, "prompt": _plain_prompt, "decode": _plain_decode,
                "sample": _plain_sample}[s["op"]](s)
    if s["op"] == "sample":
        from dequant_project_b200 import sampling
        return sampling.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                                      top_p=s["top_p"], min_p=s["min_p"])
    from dequant_project_b200 import quantized_cache as qc
    cache = qc.QuantizedCache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["k_open"], s["v_open"])
    if s["op"] == "store":
        q = qc.rope_quantized_append(s["qkv"], s["cos"], s["sin"], s["positions"], cache, s["table"], s["slots"],
                                     s["q_starts"], s["kv_lens"], s["hq"], interleaved=s["interleaved"],
                                     q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"])
        k, v, _ = qc.expanded_pages(cache, s["back_table"], s["slots"], s["back_lens"], s["back_pages"])
        return q, k, v, s["k_scale"], s["v_scale"], s["k_open"], s["v_open"]
    if s["op"] == "prompt":
        return qc.quantized_prompt_attention(s["q"], cache, s["table"], s["slots"], s["q_starts"], s["kv_lens"],
                                             s["total_pages"])
    return qc.quantized_attention(s["q"], cache, s["table"], s["slots"], s["kv_lens"])


# ---------------------------------------------------------- the definitions
def _exact_codes(x, most, codes):
    """64-bit values that rows [block, kv heads, d] stand for in 8 bits, and their scales."""
    scale = (x.abs().amax((0, 2), keepdim=True) / most).clamp(min=_LEAST)
    y = x / scale
    # e4m3: three bits behind the leading one, and steps of 2^-9 below 2^-6.
    step = 1.0 if codes == "int8" else torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale, scale[0, :, 0]


def _exact_cached(case, s, b, name):
    """64-bit rows [n, kv heads, d] of one sequence."""
    n, page, block = _numbers(case["kv_lens"])[b], case["page"], case["block"]
    done = n // block * block
    t = torch.arange(done, device="cuda")
    to, where = s["table"].long()[b, t // page], t % page
    x = s[name].float()[to, :, where].double() * s[name + "_scale"].double()[to, :, where // block][..., None]
    return torch.cat([x, s[name + "_open"][s["slots"][b], :, :n - done].transpose(0, 1).double()])


def _exact_store(case, s):
    hq, hkv, d, page, block = case["hq"], case["hkv"], case["d"], case["page"], case["block"]
    most, dtype = _CODES[case["codes"]][1], _TYPES[case["type"]]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    heads = x[:, :hq + hkv].clone()
    if case["norm"]:
        mean = (heads ** 2).sum(-1, keepdim=True) / d
        weight = torch.cat([s["q_norm"].double().expand(hq, d), s["k_norm"].double().expand(hkv, d)])
        heads = heads / torch.sqrt(mean + s["eps"]) * weight
    turned, i = heads.clone(), torch.arange(case["rot"] // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + case["rot"] // 2)
    # The angles' cosines and sines are those that the call is given.
    c, n = (s[name].double()[s["positions"]][:, None] for name in ("cos", "sin"))
    turned[..., a] = c * heads[..., a] - n * heads[..., b]
    turned[..., b] = n * heads[..., a] + c * heads[..., b]
    out = [turned[:, :hq]]
    pages, scales, opens = [], [], []
    for name, new in (("k", turned[:, hq:]), ("v", x[:, hq + hkv:])):
        new = new.to(dtype).double()  # what a 16-bit cache would hold is what is held in 8 bits
        scale, opened = s[name + "_scale"].double(), s[name + "_open"].double()
        got, at = [], 0
        for b, (q, n) in enumerate(zip(_numbers(case["q_lens"]), _numbers(case["kv_lens"]))):
            f, slot, row = _tail(case, q, n), int(s["slots"][b]), at
            at += q
            whole, first = n - n % block, (n - q) // block * block
            for t in range(f, n, block):
                to, part = int(s["table"][b, t // page]), t % page // block
                lo = max(t, n - q)  # the first new position
                if t + block <= n and q and t >= first:
                    rows = torch.cat([s[name + "_open"][slot, :, :lo - t].transpose(0, 1).double(),
                                      new[row + lo - n + q:row + t + block - n + q]])
                    rows, scale[to, :, part] = _exact_codes(rows, most, case["codes"])
                elif t + block <= n:
                    rows = s[name][to, :, t % page:t % page + block].transpose(0, 1).double() * (
                        s[name + "_scale"][to, :, part].double()[None, :, None])
                else:
                    if q and lo < n:
                        opened[slot, :, lo - whole:n - whole] = new[row + lo - n + q:row + q].transpose(0, 1)
                    rows = opened[slot, :, :n - t].transpose(0, 1)
                got.append(rows)
            got.append(torch.zeros((-(n - f) % page, hkv, d), dtype=torch.float64, device="cuda"))
        pages.append(torch.cat(got).view(-1, page, hkv, d).transpose(1, 2))
        scales.append(scale)
        opens.append(opened)
    return (*out, *pages, *scales, *opens)


def _exact_sample(s):
    """The chosen tokens are whole numbers and have no value here; what is
    given is the logarithm of the probability with which each was drawn."""
    out = []
    for r in range(s["logits"].shape[0]):
        x, heat = s["logits"][r].double(), float(s["temperature"][r])
        if heat <= 0:
            out.append(0.0)
            continue
        p = torch.softmax(x / heat, 0)
        order = torch.argsort(x, descending=True, stable=True)
        k = int(s["top_k"][r]) if s["top_k"] is not None else 0
        order = order[:k] if k > 0 else order
        if s["top_p"] is not None and float(s["top_p"][r]) < 1:
            ahead = torch.cumsum(p[order], 0)
            reach = float(s["top_p"][r]) * ahead[-1]
            order = order[:1 + int((ahead[:-1] < reach).sum())]
        if s["min_p"] is not None:
            order = order[p[order] >= float(s["min_p"][r]) * p[order[0]]]
        kept = torch.sort(order)[0]
        ahead = torch.cumsum(p[kept], 0)
        i = int((ahead <= float(s["uniform"][r]) * ahead[-1]).sum())
        out.append(float(torch.log(p[kept[min(i, len(kept) - 1)]] / ahead[-1])))
    return None, torch.tensor(out, dtype=torch.float64, device="cuda")


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return _exact_store(case, s)
    if case["op"] == "sample":
        return _exact_sample(s)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens, g, at = _numbers(case["kv_lens"]), hq // hkv, 0
    counts = _numbers(case["q_lens"]) if case["op"] == "prompt" else [1] * len(lens)
    for b, (n, c) in enumerate(zip(lens, counts)):
        if n and c:
            ends = torch.arange(n - c + 1, n + 1, device="cuda").repeat_interleave(g)
            k, v = (_exact_cached(case, s, b, name) for name in ("k", "v"))
            for h in range(hkv):
                q = s["q"][at:at + c, h * g:(h + 1) * g].double().reshape(-1, d)
                # Heads of one sequence share their mask: a few thousand rows at a time.
                for r in range(0, c * g, 8192):
                    score = q[r:r + 8192] @ k[:, h].t() * (d ** -0.5)
                    hidden = torch.arange(n, device="cuda")[None] >= ends[r:r + 8192, None]
                    p = torch.softmax(score.masked_fill(hidden, float("-inf")), 1)
                    p = p.masked_fill(hidden, 0.0).nan_to_num(0.0)
                    i = torch.arange(r, min(r + 8192, c * g), device="cuda")
                    out[at + i // g, h * g + i % g] = p @ v[:, h]
        at += c
    return out
