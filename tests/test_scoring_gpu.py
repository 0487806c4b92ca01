"""Token scores on the GPU against the numpy restatement (64 bits).

Bounds: with m the row's maximum and l its sum of exps, every term's exp is off
by a few 2^-22 and by 2^-24 of its argument (|x - m| <= 200 where it counts), the
fp32 sums round once a term along chains of at most V / 128 + 40 terms, so log l
and the entropy's two sums are relatively off by less than e = (V / 128 + 300) 2^-24:
|logprob - exact| <= e + 2^-22 |x - m|, |entropy - exact| <= 4 e (1 + exact).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def check(logits, tokens, top):
    from repercep_runtime_b200 import scoring

    got = scoring.token_logprobs(logits, tokens, top=top)
    assert got.top_ids.dtype == torch.int64 and got.top_ids.shape == (logits.shape[0], top)
    x64 = logits.double().cpu().numpy()
    V = x64.shape[1]
    e = (V / 128 + 300) * 2.0**-24
    lp, en, tl, ti = (t.cpu().numpy() for t in (got.logprobs, got.entropy, got.top_logprobs, got.top_ids))
    for r, t in enumerate(tokens.tolist()):
        ref = op.token_scores(x64[r], t, top)
        assert ti[r].tolist() == ref["ids"].tolist(), r
        for a, b in ((lp[r], ref["logprob"]), *zip(tl[r], ref["top"])):
            assert (np.isnan(a) and np.isnan(b)) or a == b or abs(a - b) <= 2 * e + 2.0**-21 * abs(b), (r, a, b)
        a, b = en[r], ref["entropy"]
        assert (np.isnan(a) and np.isnan(b)) or abs(a - b) <= 4 * e * (1 + b), (r, a, b)
    return got


def make(rows, vocab, dtype, seed=0, factor=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, vocab), generator=g) * factor).to(DTYPES[dtype])
    return x.cuda(), torch.randint(0, vocab, (rows,), generator=g).cuda()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows, vocab, top", [
    (1, 1, 1), (3, 2, 2), (2, 7, 5), (5, 127, 0), (4, 1000, 64), (2, 4097, 20), (1, 32000, 5), (3, 50001, 33),
    (300, 513, 8), (1, 160001, 1), (700, 64, 64), (9, 65536, 16),
])
def test_scores_match_the_definition(dtype, rows, vocab, top):
    x, t = make(rows, vocab, dtype, seed=vocab)
    check(x, t, top)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("offset, pitch", [(0, 1003), (1, 1001), (3, 1008), (5, 1010)])
def test_strides_and_odd_addresses(dtype, offset, pitch):
    x, t = make(6, 999, dtype, seed=pitch)
    buf = torch.full((6 * pitch + offset + 8,), float("nan"), dtype=x.dtype, device="cuda")
    view = buf[offset : offset + 6 * pitch].view(6, pitch)[:, :999]
    view.copy_(x)
    check(view, t, 7)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [33, 5000, 70000])
def test_masks_ties_and_non_finite_rows(dtype, vocab):
    x, t = make(12, vocab, dtype, seed=1)
    x[0] = float("-inf")  # nothing left
    x[1] = float("-inf")
    x[1, vocab // 2] = -4.0  # one left
    x[2, : vocab - 3] = float("-inf")  # the tail left
    x[3] = 1.5  # all equal
    x[4] = torch.finfo(x.dtype).min  # all at the type's lowest
    x[5, :] = torch.finfo(x.dtype).min
    x[5, 17] = 0.0
    x[6, 20] = float("nan")
    x[7, 21] = float("inf")
    x[8] = torch.arange(vocab, device="cuda").float().clamp(max=60000).to(x.dtype) / 64  # ascending: many equal at the end
    x[9] = 0.0
    x[9, ::2] = -0.0
    x[10] = x[10].round()
    t[10], t[11], t[1] = -1, -100, vocab // 2
    t[2] = 0  # a masked token
    check(x, t, min(vocab, 20))


def test_many_rows_and_another_stream():
    x, t = make(2000, 301, "bf16", seed=3)
    check(x, t, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(x[:40], t[:40], 3)
    torch.cuda.current_stream().wait_stream(side)


def test_offsets_past_32_bits():
    """Rows more than 2^31 elements into the tensor."""
    pitch = (1 << 30) + 8
    buf = torch.empty(2 * pitch + 4096, dtype=torch.bfloat16, device="cuda")
    view = buf.as_strided((3, 4096), (pitch, 1))
    x, t = make(3, 4096, "bf16", seed=4)
    view.copy_(x)
    check(view, t, 4)


def test_out_of_range_tokens_are_reported():
    from repercep_runtime_b200 import _lib, scoring

    x, t = make(3, 100, "fp32")
    t[1] = 100
    _lib.device_status(reset=True)
    got = scoring.token_logprobs(x, t)
    assert _lib.device_status(reset=True) == 0x203
    assert bool(got.logprobs[1].isnan()) and bool(got.logprobs[[0, 2]].isfinite().all())


def test_refusals():
    from repercep_runtime_b200 import scoring

    x, t = make(3, 100, "bf16")
    for call, words in [
        (lambda: scoring.token_logprobs(x[0], t), "2-D"),
        (lambda: scoring.token_logprobs(x.double(), t), "bf16, fp16 or fp32"),
        (lambda: scoring.token_logprobs(x.cpu(), t), "CUDA"),
        (lambda: scoring.token_logprobs(x, t.int()), "int64"),
        (lambda: scoring.token_logprobs(x, t[:2]), "int64"),
        (lambda: scoring.token_logprobs(x.t(), t), "unit-stride"),
        (lambda: scoring.token_logprobs(x, t, top=65), "top"),
        (lambda: scoring.token_logprobs(x, t, top=-1), "top"),
        (lambda: scoring.token_logprobs(x[:, :4], t, top=5), "top"),
        (lambda: scoring.token_logprobs(x[:, :0], t), "vocabulary"),
    ]:
        with pytest.raises(ValueError, match=words):
            call()
    none = scoring.token_logprobs(x[:0], t[:0], top=2)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 2)
