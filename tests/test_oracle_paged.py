"""The numpy restatement of the paged-cache operators against torch in 64 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import paged as op


def test_decode_matches_softmax_and_matmul():
    g = np.random.default_rng(0)
    q, k, v = g.standard_normal((6, 16)), g.standard_normal((2, 19, 16)), g.standard_normal((2, 19, 16))
    got = op.decode(q, k, v, 0.25)
    s = torch.einsum("hgd,hnd->hgn", torch.tensor(q).view(2, 3, 16), torch.tensor(k)) * 0.25
    p = torch.softmax(s, -1)
    np.testing.assert_allclose(got["out"], torch.einsum("hgn,hnd->hgd", p, torch.tensor(v)).reshape(6, 16), atol=1e-13)
    np.testing.assert_allclose(got["lse"], torch.logsumexp(s, -1).reshape(6), atol=1e-13)
    np.testing.assert_allclose(got["weights"], p.sum(1), atol=1e-13)
    assert np.isneginf(op.decode(q, k[:, :0], v[:, :0], 0.25)["lse"]).all()


def test_gather_rows_walks_pages():
    pool = np.arange(5 * 2 * 3).reshape(5, 2, 3)
    assert op.gather_rows(pool, np.array([4, 0, -1]), 5)[1].tolist() == [27, 28, 29, 3, 4]


@pytest.mark.parametrize("n, budget, recent", [(5, 5, 2), (9, 5, 2), (9, 5, 5), (9, 5, 0), (1, 1, 1)])
def test_kept_positions_prefer_weight_then_position(n, budget, recent):
    w = np.array([3.0, 1.0, 3.0, 0.0, 0.0, 3.0, 2.0, 9.0, 9.0])
    kept = op.kept_positions(w, n, budget, recent)
    assert len(kept) == min(n, budget) and (np.diff(kept) > 0).all()
    if n > budget:
        older = [i for i in kept if i < n - recent]
        rest = [i for i in range(n - recent) if i not in older]
        assert all((w[i], -i) > (w[j], -j) for i in older for j in rest)
    assert op.kept_positions(np.array([1.0, np.nan, 5.0, 0.0]), 4, 2, 1).tolist() == [1, 3]


def test_token_scores_match_log_softmax():
    x = np.array([0.5, -np.inf, 2.0, 2.0, -3.0])
    got = op.token_scores(x, 4, 3)
    logp = torch.log_softmax(torch.tensor(x), 0)
    assert math.isclose(got["logprob"], float(logp[4]), abs_tol=1e-14)
    assert math.isclose(got["entropy"], float(torch.special.entr(logp.exp()).sum()), abs_tol=1e-14)
    assert got["ids"].tolist() == [2, 3, 0]
    nothing = op.token_scores(np.full(4, -np.inf), 1, 2)
    assert nothing["logprob"] == -np.inf and nothing["entropy"] == 0.0 and nothing["ids"].tolist() == [0, 1]
