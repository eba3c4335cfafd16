"""Serving path over a paged cache on the GPU: ``PagedDecoder`` against
``TPDecoder.step`` token by token on the contiguous cache (whose own parity
tests pin it to an independent fp32 restatement). Both form fp16 activations
with fp32 accumulation in another order (prompts above eight rows go through
dequantize and a matrix product), so they agree to the decoder tests' 2e-3 of
the largest logit per layer pair: 5e-3 here, for GEMV against matrix product."""

from __future__ import annotations

import pytest
import torch

from decoder_reference import max_rel_err
from dequant_project_b200 import _native
from dequant_project_b200.decoder import DecoderConfig, TPDecoder
from dequant_project_b200.packer import QuantConfig
from dequant_project_b200.paged_decoder import PagedDecoder

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(n_layers=2, hidden=1024, n_heads=8, n_kv_heads=2, intermediate=2048, vocab=2000)
QCFG = QuantConfig(4, 128, False)


def one_by_one(dev, tokens):
    dec = TPDecoder(CFG, QCFG, seed=3, device=dev, batch=1, kv_len=0, max_new=len(tokens))
    return torch.cat([dec.step(tokens[i:i + 1].to(dev), i) for i in range(len(tokens))]).float()


@pytest.mark.parametrize("fuse", [True, False], ids=["swiglu-fused", "separate"])
@pytest.mark.parametrize("prefix", [0, 64])
def test_matches_the_contiguous_cache(cuda_device, prefix, fuse):
    dec = TPDecoder(CFG, QCFG, seed=3, device=cuda_device, batch=4, kv_len=0, fuse_swiglu=fuse)
    serve = PagedDecoder(dec, n_pages=64, page_size=16, max_positions=256)
    gen = torch.Generator().manual_seed(prefix)
    toks = [torch.randint(0, CFG.vocab, (n,), generator=gen) for n in (1, 16, 33, 90)]
    head = torch.randint(0, CFG.vocab, (prefix,), generator=gen)
    if prefix:
        serve.set_prefix(head)
    ids, logits = serve.add(toks)
    more = torch.randint(0, CFG.vocab, (4, 3), generator=gen)
    steps = [serve.step(ids, more[:, i]) for i in range(3)]
    for b, p in enumerate(toks):
        ref = one_by_one(cuda_device, torch.cat([head, p, more[b]]))
        n = prefix + len(p)
        assert max_rel_err(logits[b:b + 1].float(), ref[n - 1:n]) < 5e-3
        for i, s in enumerate(steps):
            assert max_rel_err(s[b:b + 1].float(), ref[n + i:n + i + 1]) < 5e-3
    assert _native.device_status(cuda_device.index) == 0


def test_more_than_eight_sequences(cuda_device):
    dec = TPDecoder(CFG, QCFG, seed=3, device=cuda_device, batch=8, kv_len=0)
    serve = PagedDecoder(dec, n_pages=64, page_size=16, max_positions=256)
    gen = torch.Generator().manual_seed(1)
    toks = [torch.randint(0, CFG.vocab, (5 + i,), generator=gen) for i in range(11)]
    ids, _ = serve.add(toks)
    nxt = torch.randint(0, CFG.vocab, (11,), generator=gen)
    got = serve.step(ids, nxt).float()
    for b in (0, 7, 10):
        ref = one_by_one(cuda_device, torch.cat([toks[b], nxt[b:b + 1]]))
        assert max_rel_err(got[b:b + 1], ref[-1:]) < 5e-3
