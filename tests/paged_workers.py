"""Worker process of the tensor-parallel serving test (spawned, one per rank).
Not a test module: pytest collects only test_*.py."""

from __future__ import annotations

import traceback

import torch


def serve(rank, world, port, queue):
    """Prompts behind a prefix and two steps; this rank's gathered logits."""
    try:
        from dequant_project_b200.decoder import DecoderConfig, TPDecoder
        from dequant_project_b200.packer import QuantConfig
        from dequant_project_b200.paged_decoder import PagedDecoder
        from tp_workers import _cpu_linear, _init

        torch.set_num_threads(2)
        dist = _init(rank, world, port, "gloo", 60) if world > 1 else None
        cfg = DecoderConfig(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, intermediate=640, vocab=1001)
        dec = TPDecoder(cfg, QuantConfig(4, 64, False), world=world, rank=rank, seed=5, batch=1, kv_len=0,
                        linear_fn=_cpu_linear)
        paged = PagedDecoder(dec, 16, 8, 64)
        gen = torch.Generator().manual_seed(2)
        tokens = torch.randint(0, cfg.vocab, (40,), generator=gen)
        paged.set_prefix(tokens[:8])
        ids, first = paged.add([tokens[8:11], tokens[11:30]])
        out = [first, paged.step(ids, tokens[30:32]), paged.step(ids[::-1], tokens[32:34])]
        queue.put((rank, torch.stack(out).float().numpy(), None))
        if dist is not None:
            dist.barrier()
            dist.destroy_process_group()
    except Exception:  # reported to the test, which fails with it
        queue.put((rank, None, traceback.format_exc()))


def serve_quantized(rank, world, port, queue):
    """The same over an 8-bit cache, and tokens drawn with a generator that all
    ranks have seeded alike; this rank's logits and tokens."""
    try:
        from dequant_project_b200.decoder import DecoderConfig, TPDecoder
        from dequant_project_b200.packer import QuantConfig
        from dequant_project_b200.paged_decoder import PagedDecoder
        from tp_workers import _cpu_linear, _init

        torch.set_num_threads(2)
        dist = _init(rank, world, port, "gloo", 60) if world > 1 else None
        cfg = DecoderConfig(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, intermediate=640, vocab=1001)
        dec = TPDecoder(cfg, QuantConfig(4, 64, False), world=world, rank=rank, seed=5, batch=1, kv_len=0,
                        linear_fn=_cpu_linear)
        paged = PagedDecoder(dec, 16, 16, 96, codes=torch.int8, max_seqs=2)
        gen = torch.Generator().manual_seed(2)
        tokens = torch.randint(0, cfg.vocab, (80,), generator=gen)
        paged.set_prefix(tokens[:16])
        ids, first = paged.add([tokens[16:19], tokens[19:50]])  # the steps complete a block of each
        out = [first, *(paged.step(ids[::1 - 2 * (i % 2)], tokens[50 + 2 * i:52 + 2 * i]) for i in range(14))]
        for i in ids:
            paged.free(i)
        draws = paged.generate([tokens[:5], tokens[5:30]], 8, torch.Generator().manual_seed(7), temperature=1.3, top_p=0.9)
        queue.put((rank, (torch.stack(out).float().numpy(), draws.numpy()), None))
        if dist is not None:
            dist.barrier()
            dist.destroy_process_group()
    except Exception:  # reported to the test, which fails with it
        queue.put((rank, None, traceback.format_exc()))
