"""Serving path of the packed decoder: prompts in, then decode steps, for
sequences of different lengths over a paged key/value cache.

``TPDecoder.step`` decodes sequences that share one length on a contiguous
cache that something else has filled. ``PagedDecoder`` takes a ``TPDecoder``'s
packed weights and runs them over pages (``paged_ops``): ``add`` runs packed
prompts of any lengths through every layer at once (``rope_paged_append``, then
``prompt_attention``), ``step`` decodes one token of every sequence
(``paged_attention``, or ``shared_prefix_attention`` where the sequences begin
with the prefix that ``set_prefix`` has cached once), ``free`` returns a
sequence's pages, ``sample`` draws the next tokens (``sample_tokens``). With
``codes`` the cache is held in 8 bits (``quantized_cache``: half the bytes a
decode step reads, twice the positions in the same memory). Linear layers go
through the fused GEMV up to eight rows and through dequantize and a matrix
product above, as ``QuantLinear`` does.

The reference models the decode step's bytes
(KrishnaI2424/Dequant_Project ``dequant/byte_model.py:179-251``) and has no
prompt or cache code.

    python -m dequant_project_b200.paged_decoder --seqs 8 --prompt 300 --steps 32

runs a random-weight model on one GPU and prints its rates.
"""

from __future__ import annotations

import torch

from dequant_project_b200 import decode_ops as ops
from dequant_project_b200 import paged_ops as paged
from dequant_project_b200 import quantized_cache as quantized
from dequant_project_b200.decoder import TPDecoder
from dequant_project_b200.sampling import sample_tokens


class PageAllocator:
    """Page numbers of a pool (or other things' numbers), handed out and taken
    back on the host."""

    def __init__(self, n_pages: int, what: str = "pages"):
        self.free = list(range(n_pages - 1, -1, -1))
        self.what = what

    def take(self, n: int) -> list[int]:
        if n > len(self.free):
            raise RuntimeError(f"{n} {self.what} needed, {len(self.free)} free")
        got = self.free[len(self.free) - n:][::-1]
        del self.free[len(self.free) - n:]
        return got

    def give(self, pages: list[int]) -> None:
        self.free.extend(reversed(pages))


class PagedDecoder:
    """A decoder's weights over a paged cache of ``n_pages`` pages a layer
    (this rank's heads), ``page_size`` positions each, for sequences of up to
    ``max_positions`` positions. ``codes`` (int8 or float8_e4m3fn; default: 16
    bits) holds the cache in 8 bits, with a scale for every ``block`` positions
    of a head and open blocks for ``max_seqs`` sequences (4 * block * head_dim
    bytes a head of keys and values, layer and sequence). A pass over prompts then
    takes scratch memory of 4 * head_dim bytes a head for every position that its
    sequences have, twice what the codes take; and a prefix is shared in the pages
    alone: ``add`` expands it, and ``step`` reads it, once for every sequence, where
    the 16-bit cache's is read once a batch. At world > 1 every rank makes the same
    calls."""

    def __init__(self, dec: TPDecoder, n_pages: int, page_size: int = 16, max_positions: int = 4096,
                 rope_scaling: dict | None = None, *, codes: torch.dtype | None = None, block: int = 16,
                 max_seqs: int = 64):
        cfg = dec.cfg
        self.dec, self.page, self.max_positions = dec, page_size, max_positions
        self.codes = codes
        if codes is None:
            shape = (n_pages, dec.hkv, page_size, cfg.head_dim)
            self.k = [torch.zeros(shape, dtype=torch.float16, device=dec.device) for _ in range(cfg.n_layers)]
            self.v = [torch.zeros(shape, dtype=torch.float16, device=dec.device) for _ in range(cfg.n_layers)]
        else:
            # (One open block more than sequences: a prefix passes through it.)
            self.cache = [quantized.QuantizedCache.empty(n_pages, dec.hkv, page_size, cfg.head_dim, max_seqs + 1,
                                                         block=block, codes=codes, device=dec.device)
                          for _ in range(cfg.n_layers)]
            self.open = PageAllocator(max_seqs, "open blocks")
        self.cos, self.sin = paged.rope_scaled_tables(cfg.head_dim, cfg.rope_theta, max_positions, dec.device,
                                                      scaling=rope_scaling)
        self.pages = PageAllocator(n_pages)
        self.seqs: dict[int, dict] = {}  # id -> own pages, own length (and open block)
        self.prefix_pages: list[int] = []
        self.prefix_len = 0
        self._next = 0

    # ------------------------------------------------------------- the layers
    def _linear(self, x: torch.Tensor, pw) -> torch.Tensor:
        return self.dec._linear(x, pw)

    def _reduce(self, t: torch.Tensor) -> torch.Tensor:
        if self.dec.world > 1:
            import torch.distributed as dist
            dist.all_reduce(t, op=dist.ReduceOp.SUM, group=self.dec.group)
        return t

    def _mlp(self, x: torch.Tensor, gu) -> torch.Tensor:
        dec = self.dec
        if dec.gu_order is None:
            return ops.silu_mul(self._linear(x, gu))
        from dequant_project_b200.quant_linear import _format_args
        bits, gs, _, _ = _format_args(gu.config, x.shape[1])
        if x.shape[0] <= 8 and ops.gemv_swiglu_supported(x.shape[0], gu.shape[0], x.shape[1], bits, gs):
            return ops.gemv_swiglu(x, gu)
        # Gate and up rows are stored interleaved by eights (gate_up_order).
        both = self._linear(x, gu).view(x.shape[0], -1, 2, 8)
        return ops.silu_mul(both.transpose(1, 2).reshape(x.shape[0], -1))

    def _embed(self, tokens: torch.Tensor) -> torch.Tensor:
        """Rows of the embedding. A token below 0, which ``sample`` draws from
        logits that are not numbers, is NaN, not another token's row: its sequence's
        logits are not numbers either, and its further draws -1."""
        if not tokens.is_cuda:
            return self.dec.embed[tokens]
        h = self.dec.embed[tokens.clamp(min=0)]
        return h.masked_fill_((tokens < 0)[:, None], float("nan"))

    def _forward(self, tokens, store, attend, last) -> torch.Tensor:
        """All layers over packed tokens: ``store(layer, qkv)`` rotates, puts
        keys and values into the cache and gives the queries, ``attend(layer,
        q)`` is the attention. Logits of rows ``last``."""
        dec, cfg = self.dec, self.dec.cfg
        h = self._embed(tokens)
        pending = None
        for layer, w in enumerate(dec.layers):
            x = ops.add_rms_norm(h, pending, dec.attn_norm[layer], cfg.eps)
            a = attend(layer, store(layer, self._linear(x, w["qkv"]))).reshape(tokens.shape[0], -1)
            x = ops.add_rms_norm(h, self._reduce(self._linear(a, w["o"])), dec.mlp_norm[layer], cfg.eps)
            pending = self._reduce(self._linear(self._mlp(x, w["gu"]), w["down"]))
        x = ops.add_rms_norm(h, pending, dec.final_norm, cfg.eps)[last].contiguous()
        logits = dec._lm_head(x)
        if dec.world == 1:
            return logits
        import torch.distributed as dist
        bounds = dec.vocab_bounds
        width = max(b - a for a, b in zip(bounds[:-1], bounds[1:]))
        padded = logits.new_zeros((logits.shape[0], width))
        padded[:, :logits.shape[1]] = logits
        parts = [torch.empty_like(padded) for _ in range(dec.world)]
        dist.all_gather(parts, padded, group=dec.group)
        return torch.cat([p[:, :b - a] for p, a, b in zip(parts, bounds[:-1], bounds[1:])], dim=1)

    def _ints(self, values, dtype=torch.int32) -> torch.Tensor:
        return torch.tensor(values, dtype=dtype).to(self.dec.device, non_blocking=True)

    def _table(self, rows: list[list[int]]) -> torch.Tensor:
        width = max(1, max(len(r) for r in rows))
        return self._ints([r + [0] * (width - len(r)) for r in rows])

    def _slots(self, pages: list[int], start: int, n: int) -> list[int]:
        return [pages[t // self.page] * self.page + t % self.page for t in range(start, start + n)]

    def _store(self, positions, slots):
        """What puts tokens into 16-bit pages, at ``slots``."""
        def store(layer, qkv):
            return paged.rope_paged_append(qkv, self.cos, self.sin, positions, slots, self.k[layer], self.v[layer],
                                           self.dec.hq)
        return store

    def _store_quantized(self, positions, table, open_slots, q_starts, kv_lens):
        """What puts tokens into 8-bit pages, as the newest of the sequences."""
        def store(layer, qkv):
            return quantized.rope_quantized_append(qkv, self.cos, self.sin, positions, self.cache[layer], table,
                                                   open_slots, q_starts, kv_lens, self.dec.hq)
        return store

    def _prompts(self, prompts, tables, starts, opens) -> torch.Tensor:
        """Packed prompts whose rows continue cached sequences: ``tables`` their
        pages, ``starts`` the positions already cached, ``opens`` their open
        blocks."""
        lens = [int(p.shape[0]) for p in prompts]
        ends = [s + n for s, n in zip(starts, lens)]
        bounds = [0]
        for n in lens:
            bounds.append(bounds[-1] + n)
        positions = self._ints([t for s, e in zip(starts, ends) for t in range(s, e)], torch.int64)
        table, q_starts, kv_lens = self._table(tables), self._ints(bounds), self._ints(ends)
        if self.codes is None:
            store = self._store(positions, self._ints([t for pages, s, n in zip(tables, starts, lens)
                                                       for t in self._slots(pages, s, n)], torch.int64))

            def attend(layer, q):
                return paged.prompt_attention(q, self.k[layer], self.v[layer], table, q_starts, kv_lens)
        else:
            open_slots, n_pages = self._ints(opens), sum(-(-n // self.page) for n in ends)
            store = self._store_quantized(positions, table, open_slots, q_starts, kv_lens)

            def attend(layer, q):
                return quantized.quantized_prompt_attention(q, self.cache[layer], table, open_slots, q_starts, kv_lens,
                                                            n_pages)

        tokens = torch.cat([p.to(self.dec.device) for p in prompts])
        return self._forward(tokens, store, attend, self._ints([b - 1 for b in bounds[1:]], torch.int64))

    def _take_open(self, n: int) -> list[int]:
        return [0] * n if self.codes is None else self.open.take(n)

    def _give_open(self, opens: list[int]) -> None:
        if self.codes is not None:
            self.open.give(opens)

    def _check_tokens(self, tokens: torch.Tensor) -> None:
        """Tokens on the host are looked at: one outside the vocabulary would be
        another token's row (negative) or a fault on the GPU. (Those on the GPU
        come from logits, and looking at them would wait for it.)"""
        if not tokens.is_cuda and tokens.numel():
            lo, hi = int(tokens.min()), int(tokens.max())
            if lo < 0 or hi >= self.dec.cfg.vocab:
                raise ValueError(f"tokens must be in [0, {self.dec.cfg.vocab}), got {lo if lo < 0 else hi}")

    # ------------------------------------------------------------- the calls
    def set_prefix(self, tokens: torch.Tensor) -> None:
        """Cache ``tokens`` once as the beginning of every sequence added from
        now on (a whole number of pages; before any sequence)."""
        n = int(tokens.shape[0])
        if self.seqs or self.prefix_len:
            raise RuntimeError("the prefix is set once, before any sequence is added")
        if n < 1 or n % self.page or n >= self.max_positions:
            raise ValueError(f"a prefix holds whole pages of {self.page} and leaves room in "
                             f"{self.max_positions} positions, got {n}")
        self._check_tokens(tokens)
        pages = self.pages.take(n // self.page)
        try:
            self._prompts([tokens], [pages], [0], [len(self.open.free)] if self.codes is not None else [0])
        except BaseException:
            self.pages.give(pages)
            raise
        self.prefix_pages, self.prefix_len = pages, n

    def add(self, prompts: list[torch.Tensor]) -> tuple[list[int], torch.Tensor]:
        """Run new sequences' prompts (int64, at least one token each) in one
        packed pass. Returns their ids and their last tokens' logits. A pass
        that raises adds nothing."""
        for p in prompts:
            if p.dim() != 1 or p.shape[0] < 1 or self.prefix_len + p.shape[0] > self.max_positions:
                raise ValueError(f"a prompt holds 1 to {self.max_positions - self.prefix_len} tokens")
            self._check_tokens(p)
        taken: list[list[int]] = []
        opens = self._take_open(len(prompts))
        try:
            for p in prompts:
                taken.append(self.pages.take(-(-int(p.shape[0]) // self.page)))
            logits = self._prompts(prompts, [self.prefix_pages + t for t in taken], [self.prefix_len] * len(prompts),
                                   opens)
        except BaseException:
            for t in reversed(taken):
                self.pages.give(t)
            self._give_open(opens)
            raise
        ids = []
        for p, t, o in zip(prompts, taken, opens):
            self.seqs[self._next] = {"pages": t, "len": int(p.shape[0]), "open": o}
            ids.append(self._next)
            self._next += 1
        return ids, logits

    def step(self, ids: list[int], tokens: torch.Tensor) -> torch.Tensor:
        """One token of each of the sequences ``ids`` (int64 [len(ids)]): its
        logits [len(ids), vocab]. A step that raises leaves the sequences as
        they were, so that it can be taken again."""
        if tokens.shape != (len(ids),) or len(set(ids)) != len(ids):
            raise ValueError("step takes one token for each of different sequences")
        self._check_tokens(tokens)
        seqs = [self.seqs[i] for i in ids]
        for s in seqs:
            if self.prefix_len + s["len"] >= self.max_positions:
                raise ValueError(f"a sequence has reached {self.max_positions} positions")
        short = [s for s in seqs if s["len"] == len(s["pages"]) * self.page]
        more = self.pages.take(len(short))
        for s, page in zip(short, more):
            s["pages"].append(page)
        try:
            logits = self._step(seqs, tokens)
        except BaseException:
            for s in short:
                s["pages"].pop()
            self.pages.give(more)
            raise
        for s in seqs:
            s["len"] += 1
        return logits

    def _step(self, seqs: list[dict], tokens: torch.Tensor) -> torch.Tensor:
        positions = self._ints([self.prefix_len + s["len"] for s in seqs], torch.int64)
        if self.codes is not None:
            # (The prefix is read as every sequence's own beginning.)
            table = self._table([self.prefix_pages + s["pages"] for s in seqs])
            lens = self._ints([self.prefix_len + s["len"] + 1 for s in seqs])
            open_slots, starts = self._ints([s["open"] for s in seqs]), self._ints(range(len(seqs) + 1))

            def attend(layer, q):
                return quantized.quantized_attention(q, self.cache[layer], table, open_slots, lens)

            return self._forward(tokens.to(self.dec.device),
                                 self._store_quantized(positions, table, open_slots, starts, lens), attend, slice(None))
        store = self._store(positions, self._ints([self._slots(s["pages"], s["len"], 1)[0] for s in seqs], torch.int64))
        table, lens = self._table([s["pages"] for s in seqs]), self._ints([s["len"] + 1 for s in seqs])
        if self.prefix_len:
            prefix = self._ints(self.prefix_pages)

            def attend(layer, q):
                return paged.shared_prefix_attention(q, self.k[layer], self.v[layer], prefix, self.prefix_len,
                                                     table, lens)
        else:
            def attend(layer, q):
                return paged.paged_attention(q, self.k[layer], self.v[layer], table, lens)
        return self._forward(tokens.to(self.dec.device), store, attend, slice(None))

    def free(self, seq: int) -> None:
        """Forget a sequence and return its pages."""
        s = self.seqs.pop(seq)
        self.pages.give(s["pages"])
        self._give_open([s["open"]])

    def sample(self, logits: torch.Tensor, generator: torch.Generator | None = None, **params) -> torch.Tensor:
        """The next tokens of rows of logits: ``sample_tokens`` with ``params``
        (temperature, top_k, top_p, min_p) and random numbers of ``generator``
        (of the model's device; at world > 1 one is needed that every rank has
        seeded alike). Without params the largest logits. A row without a logit
        above -inf draws -1: ``step`` takes that on the GPU as a token of no
        value (the sequence's logits become NaN), and refuses it on the host."""
        if not params:
            return logits.argmax(-1)
        if self.dec.world > 1 and generator is None:
            raise ValueError("sampling on several ranks needs a generator that all have seeded alike")
        uniform = torch.rand(logits.shape[0], generator=generator, device=logits.device)
        return sample_tokens(logits, uniform, **params)[0]

    def generate(self, prompts: list[torch.Tensor], steps: int, generator: torch.Generator | None = None,
                 **params) -> torch.Tensor:
        """The prompts' next ``steps`` tokens, [len(prompts), steps]: greedy, or
        drawn as ``sample`` draws them."""
        if steps < 1:
            return torch.empty((len(prompts), 0), dtype=torch.int64, device=self.dec.device)
        ids, logits = self.add(prompts)
        try:
            out = [self.sample(logits, generator, **params)]
            while len(out) < steps:
                out.append(self.sample(self.step(ids, out[-1]), generator, **params))
        finally:
            for i in ids:
                self.free(i)
        return torch.stack(out, 1)


def main() -> None:
    import argparse
    import time

    from dequant_project_b200 import decoder as D
    from dequant_project_b200.packer import QuantConfig

    ap = argparse.ArgumentParser(description="Prompts and decode steps of a random-weight packed decoder.")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--seqs", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=300, help="longest prompt; the others are shorter")
    ap.add_argument("--prefix", type=int, default=0, help="tokens that all sequences share (whole pages)")
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--page", type=int, default=16)
    ap.add_argument("--cache", choices=("fp16", "int8", "e4m3"), default="fp16")
    ap.add_argument("--temperature", type=float, default=0.0, help="0: the largest logit")
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    args = ap.parse_args()
    base = D.LLAMA2_7B
    cfg = D.DecoderConfig(args.layers, base.hidden, base.n_heads, base.n_kv_heads, base.intermediate, base.vocab)
    dec = TPDecoder(cfg, QuantConfig(4, 128, False), device="cuda", kv_len=0, batch=min(args.seqs, 8))
    longest = args.prefix + args.prompt + args.steps
    pages = args.seqs * -(-(args.prompt + args.steps) // args.page) + args.prefix // args.page
    serve = PagedDecoder(dec, pages, args.page, longest, max_seqs=args.seqs,
                         codes={"fp16": None, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}[args.cache])
    params = {} if args.temperature == 0 else dict(temperature=args.temperature, top_k=args.top_k, top_p=args.top_p,
                                                   min_p=args.min_p)
    gen = torch.Generator().manual_seed(0)
    if args.prefix:
        serve.set_prefix(torch.randint(0, cfg.vocab, (args.prefix,), generator=gen))
    prompts = [torch.randint(0, cfg.vocab, (max(1, args.prompt * (i + 1) // args.seqs),), generator=gen)
               for i in range(args.seqs)]
    serve.generate(prompts, 2, **params)  # warm-up
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    ids, logits = serve.add(prompts)
    torch.cuda.synchronize()
    t1 = time.perf_counter()
    for _ in range(args.steps):
        logits = serve.step(ids, serve.sample(logits, **params))
    torch.cuda.synchronize()
    t2 = time.perf_counter()
    total = sum(int(p.shape[0]) for p in prompts)
    print(f"{cfg.n_layers} layers, {args.seqs} sequences: prompts {total} tokens in {1e3 * (t1 - t0):.2f} ms, "
          f"{args.steps} steps at {1e3 * (t2 - t1) / args.steps:.2f} ms")


if __name__ == "__main__":
    main()
