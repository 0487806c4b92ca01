"""The element-wise bounds on a decode's rounding errors let through what the
operator rounds, and not a weight rounded once or a weight lost below fp16's
range (mistakes planted in a numpy restatement)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as op

FORMATS = {"bf16": (torch.bfloat16, 2.0**-8), "fp16": (torch.float16, 2.0**-11)}


def rounded(x, fmt):
    return torch.tensor(x).to(FORMATS[fmt][0]).double().numpy()


def restated(q, k, v, scale, fmt, parts, top):
    """A decode whose weights, 2^top at the largest, enter their product in
    ``parts`` values of the format ``fmt``."""
    H = k.shape[0]
    s = np.einsum("hgd,hnd->hgn", q.reshape(H, -1, q.shape[1]), k) * scale
    e = np.exp(s - s.max(-1, keepdims=True))
    used, rest = np.zeros_like(e), e * 2.0**top
    for _ in range(parts):
        part = rounded(rest, fmt)
        used, rest = used + part, rest - part
    out = np.einsum("hgn,hnd->hgd", used / (e.sum(-1, keepdims=True) * 2.0**top), v)
    return rounded(out.reshape(q.shape), fmt)


@pytest.mark.parametrize("fmt", ["bf16", "fp16"])
def test_a_weight_rounded_once_is_beyond_the_bound_of_two_parts(fmt):
    """Few keys and small scores, so that the bound is little more than the
    output's rounding where the values cancel."""
    g = np.random.default_rng(1)
    q, k, v = (rounded(f * g.standard_normal(s), fmt) for f, s in ((0.5, (32, 64)), (1.0, (2, 6, 64)), (1.0, (2, 6, 64))))
    u = FORMATS[fmt][1]
    exact = op.decode(q, k, v, 0.125)["out"]
    bound = op.decode_bound(q, k, v, 0.125, u, u * u, np.zeros((32, 6)))["out"]
    assert (np.abs(restated(q, k, v, 0.125, fmt, 2, 0) - exact) <= bound).all()
    assert (np.abs(restated(q, k, v, 0.125, fmt, 1, 0) - exact) > bound).any()


def test_weights_below_fp16s_range_are_beyond_the_bound():
    """One dominant key, the others 2^-26 of it: at the top of fp16's range they
    are held, at 1 they are gone."""
    g = np.random.default_rng(2)
    q = np.ones((1, 64))
    k = np.zeros((1, 400, 64))
    k[0, 7] = 26 * np.log(2.0) / 64
    v = rounded(30000.0 * (1 + 0.1 * g.standard_normal((1, 400, 64))), "fp16")
    v[0, 7] = 0.0
    p = np.exp((k[0] @ q[0]) - 26 * np.log(2.0))
    floor = np.full((1, 400), 2.0**-36) * p.max() / p.sum()
    exact = op.decode(q, k, v, 1.0)["out"]
    bound = op.decode_bound(q, k, v, 1.0, 2.0**-11, 2.0**-22, floor)["out"]
    assert (np.abs(restated(q, k, v, 1.0, "fp16", 2, 11) - exact) <= bound).all()
    assert (np.abs(restated(q, k, v, 1.0, "fp16", 2, 0) - exact) > bound).all()
