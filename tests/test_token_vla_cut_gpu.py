"""The candidate-decoding example with a cut prompt against a dense fp32
decoder: the observed attention weights, what stays of the prompt, and the
candidates' log probabilities over it."""

from __future__ import annotations

import pytest
import torch
from test_token_vla_example_gpu import example  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_heads", [2, 8])
def test_a_cut_prompt_matches_a_dense_decoder(example, kv_heads, monkeypatch):  # noqa: F811
    from repercep_runtime_b200 import _lib, paged

    _lib.device_status(reset=True)
    cfg = example.Config(layers=1, heads=8, kv_heads=kv_heads, head_dim=64, hidden=256, vocab=500, page=16)
    model = example.Decoder(cfg)
    # the last tokens repeat a few ids, so that they attend to each other
    prompt = torch.randint(0, cfg.vocab, (192,), generator=torch.Generator().manual_seed(3)).cuda()
    observe, budget = 24, 64
    prompt[-observe:] = prompt[-observe:][torch.arange(observe) % 3]
    seen = {}
    evict = paged.evict

    def spy(cache, table, lengths, weights, out_table, **kw):
        seen["weights"] = weights.clone()
        return evict(cache, table, lengths, weights, out_table, **kw)

    monkeypatch.setattr(example.paged, "evict", spy)
    got = example.plan(model, prompt, candidates=5, steps=12, budget=budget, observe=observe)
    P, G, D = prompt.shape[0], cfg.heads // kv_heads, cfg.head_dim
    q, k, v = (t.double() for t in model.project(0, model.embed[prompt]))
    s = torch.einsum("thgd,jhd->hgtj", q[-observe:].view(observe, kv_heads, G, D), k) / D**0.5
    ahead = torch.arange(P, device="cuda") > torch.arange(P - observe, P, device="cuda").view(-1, 1)
    weights = torch.softmax(s.masked_fill(ahead, float("-inf")), -1).sum((1, 2))  # (kv_heads, P)
    # the projections here round as the example's do; scores are within 2^-10 in fp32
    assert bool(((seen["weights"][0, :, :P] - weights).abs() <= 2.0**-8 * weights + 1e-6).all())

    kept = got.kept[0].long()
    assert bool((kept[:, -observe:] == torch.arange(P - observe, P, device="cuda")).all())
    for h in range(kv_heads):
        older = kept[h, : budget - observe]
        gone = torch.ones(P - observe, dtype=torch.bool, device="cuda")
        gone[older] = False
        assert float(weights[h, older].min()) >= (1 - 2.0**-7) * float(weights[h, : P - observe][gone].max())

    # candidates: a step's attention is over the kept prompt rows and the candidate's own
    model32 = [w.float() for w in (model.qkv[0], model.out[0], model.head)]

    def project(x):
        y = (x @ model32[0]).view(x.shape[0], cfg.heads + 2 * kv_heads, D)
        return y[:, : cfg.heads], y[:, cfg.heads : cfg.heads + kv_heads], y[:, cfg.heads + kv_heads :]

    def attend(qx, kx, vx):
        """(heads, D) and (kv_heads, n, D) to (heads * D,)."""
        sx = torch.einsum("hgd,hnd->hgn", qx.view(kv_heads, G, D), kx) / D**0.5
        return torch.einsum("hgn,hnd->hgd", torch.softmax(sx, -1), vx).reshape(-1)

    x = model.embed[prompt].float()
    pq, pk, pv = project(x)
    last = x[-1] + attend(pq[-1], pk.transpose(0, 1), pv.transpose(0, 1)) @ model32[1]
    worst = 0.0
    for c in range(5):
        logits = last @ model32[2]
        keys = torch.stack([pk[kept[h], h] for h in range(kv_heads)])
        vals = torch.stack([pv[kept[h], h] for h in range(kv_heads)])
        for step, token in enumerate(got.tokens[c].tolist()):
            worst = max(worst, abs(float(torch.log_softmax(logits, -1)[token] - got.logprobs[c, step])))
            h0 = model.embed[token].float()
            cq, ck, cv = project(h0[None])
            keys, vals = torch.cat([keys, ck.transpose(0, 1)], 1), torch.cat([vals, cv.transpose(0, 1)], 1)
            logits = (h0 + attend(cq[0], keys, vals) @ model32[1]) @ model32[2]
    # bf16 activations and an FP8 prompt attention against fp32, as for an uncut prompt
    assert worst < 0.25, worst
    assert _lib.device_status() == 0
