"""The candidate-decoding example (paged append, decode, evict and token
scores together) against a dense fp32 decoder that sees the same tokens."""

from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "token_vla_decode.py"
    spec = importlib.util.spec_from_file_location("token_vla_decode", path)
    module = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = module
    spec.loader.exec_module(module)
    return module


def dense_logprobs(model, prompt, tokens):
    """Log probabilities of one candidate's tokens: plain fp32 attention over
    the whole sequence (weights and projections as the example has them)."""
    c = model.cfg
    ids = torch.cat([prompt, tokens])
    x = model.embed[ids].float()
    n, group = ids.shape[0], c.heads // c.kv_heads
    mask = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
    for layer in range(c.layers):
        y = (x @ model.qkv[layer].float()).view(n, -1, c.head_dim)
        q, k, v = y[:, : c.heads], y[:, c.heads : c.heads + c.kv_heads], y[:, c.heads + c.kv_heads :]
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        s = torch.einsum("qhd,khd->hqk", q, k) / c.head_dim**0.5
        p = torch.softmax(s.masked_fill(~mask, float("-inf")), -1)
        x = x + torch.einsum("hqk,khd->qhd", p, v).reshape(n, -1) @ model.out[layer].float()
    logits = x[prompt.shape[0] - 1 : -1] @ model.head.float()
    return torch.log_softmax(logits, -1).gather(1, tokens.view(-1, 1)).view(-1)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("kv_heads", [2, 8])
def test_plan_matches_a_dense_decoder(example, kv, kv_heads):
    from repercep_runtime_b200 import _lib, paged

    _lib.device_status(reset=True)
    cfg = example.Config(layers=2, heads=8, kv_heads=kv_heads, head_dim=64, hidden=256, vocab=1000, page=16)
    model = example.Decoder(cfg)
    prompt = torch.randint(0, cfg.vocab, (160,), generator=torch.Generator().manual_seed(1)).cuda()
    dtype = torch.bfloat16 if kv == "bf16" else paged.FP8
    got = example.plan(model, prompt, candidates=6, steps=20, kv=dtype)
    assert got.tokens.shape == (6, 20) and got.best == int(got.logprobs.sum(1).argmax())
    worst = max(float((dense_logprobs(model, prompt, got.tokens[i]) - got.logprobs[i]).abs().max()) for i in range(6))
    # bf16 activations (8 bits) and an FP8 prompt attention (4 bits a value, averaged over
    # the keys) against fp32: logits of standard deviation 2 that move by a few per cent
    assert worst < 0.25, worst
    assert _lib.device_status() == 0


def test_plan_with_a_cut_prompt(example):
    from repercep_runtime_b200 import _lib

    _lib.device_status(reset=True)
    cfg = example.Config(layers=2, heads=8, kv_heads=4, head_dim=64, hidden=256, vocab=1000, page=16)
    model = example.Decoder(cfg)
    prompt = torch.randint(0, cfg.vocab, (320,), generator=torch.Generator().manual_seed(2)).cuda()
    got = example.plan(model, prompt, candidates=3, steps=5, budget=128, observe=8)
    assert got.kept.shape == (1, 4, 128)
    assert bool((got.kept[:, :, -8:] == torch.arange(312, 320, device="cuda")).all())
    assert bool((got.kept.diff(dim=-1) > 0).all())
    assert bool(got.logprobs.isfinite().all()) and bool((got.logprobs <= 0).all())
    assert _lib.device_status() == 0
    with pytest.raises(ValueError, match="pages"):
        example.plan(model, prompt, candidates=3, steps=5, budget=100)
