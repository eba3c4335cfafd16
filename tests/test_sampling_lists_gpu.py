"""Draws whose candidates fill some CTAs' lists of a row and not others': the cut
of top-k from the threads' largest logits, with as many tokens above it as a list
holds, and then top-p. Against the 64-bit restatement, as in test_sampling_gpu.py."""

from __future__ import annotations

import pytest
import torch

from test_sampling_gpu import compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,dtype", [(160, 32768, torch.float32), (40, 131072, torch.float16),
                                              (20, 65536, torch.bfloat16), (150, 16384, torch.float32)], ids=str)
@pytest.mark.parametrize("share", [0.5, 0.9, 0.97, 0.98, 0.99, 1.0, 1.5])
def test_lists_about_full(cuda_device, rows, vocab, dtype, share):
    """``share``: top_k over the number of threads (512 for every 16384 tokens in
    fp32, 32768 in 16 bits)."""
    gen = torch.Generator(device=cuda_device).manual_seed(int(100 * share))
    top_k = int(share * 512 * vocab / (16384 if dtype == torch.float32 else 32768))
    logits = (3 * torch.randn((rows, vocab), generator=gen, device=cuda_device)).to(dtype)
    uniform = torch.rand(rows, generator=gen, device=cuda_device)
    top_p = torch.rand(rows, generator=gen, device=cuda_device)
    compare(logits, uniform, top_k=top_k, top_p=top_p, temperature=1.5)
    compare(logits, uniform, top_k=top_k, top_p=0.9999)
    compare(logits, uniform, top_k=top_k, temperature=30.0)


@pytest.mark.parametrize("skew", [0.0, 2.0, 8.0])
def test_candidates_in_one_part_of_the_row(cuda_device, skew):
    """One CTA's tokens lie above the others', so that only its list overflows."""
    gen = torch.Generator(device=cuda_device).manual_seed(9)
    logits = torch.randn((30, 100000), generator=gen, device=cuda_device)
    logits[:, 30000:60000] += skew
    uniform = torch.rand(30, generator=gen, device=cuda_device)
    for params in (dict(top_p=0.3), dict(top_p=0.9, temperature=0.5), dict(top_k=1500, top_p=0.7),
                   dict(top_k=3000, top_p=0.95, min_p=0.01), dict(top_k=40000)):
        compare(logits, uniform, **params)


@pytest.mark.parametrize("rows,vocab,dtype", [(64, 128256, torch.float16), (40, 131072, torch.bfloat16),
                                              (150, 16384, torch.float32), (160, 32768, torch.float32)], ids=str)
@pytest.mark.parametrize("top_p", [0.05, 0.5, 0.9])
def test_a_list_for_top_p_where_top_k_has_overflowed(cuda_device, rows, vocab, dtype, top_p):
    """top_k of nearly as many tokens as there are threads, some of which have but
    unlikely tokens, so that no list holds the candidates; and few tokens that have
    top_p of the sum."""
    gen = torch.Generator(device=cuda_device).manual_seed(rows)
    threads = 512 * -(-vocab // (16384 if dtype == torch.float32 else 32768))
    logits = (3 * torch.randn((rows, vocab), generator=gen, device=cuda_device)).abs().to(dtype)
    size = logits.element_size()
    # (What five threads of a CTA read: of every 8192 bytes 16 each.)
    logits[:, torch.arange(vocab, device=cuda_device) % (8192 // size) < 80 // size] = 2.0
    logits[::3] = torch.round(logits[::3])  # ties, thousands at the cut
    uniform = torch.rand(rows, generator=gen, device=cuda_device)
    for params in (dict(), dict(temperature=0.5), dict(temperature=2.0, min_p=0.01)):
        compare(logits, uniform, top_k=threads - 3, top_p=top_p, **params)
