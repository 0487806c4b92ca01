"""Paged-cache attention, eviction and token scores in numpy, 64 bits.  Test
infrastructure only.

No reference code stands behind these (the reference keeps its decode cache in
HF ``generate``, scripts/run_vla_openvla_gpu.py:174-186): the formulas are the
definition.
"""

from __future__ import annotations

import numpy as np


def gather_rows(pool: np.ndarray, table_row: np.ndarray, n: int) -> np.ndarray:
    """(heads, n, ...) rows of one sequence from a (pages, heads, page, ...) pool."""
    page = pool.shape[2]
    pos = np.arange(n)
    return np.moveaxis(pool[np.asarray(table_row, dtype=np.int64)[pos // page], :, pos % page], 0, 1)


def decode(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float) -> dict[str, np.ndarray]:
    """One sequence: q (Hq, D), k / v (H, n, D) in float64.

    ``out``, ``lse``, ``weights`` (H, n; summed over the group), and what a
    bound on rounding errors needs: ``abs_out`` = sum_j p_j |v_j| and
    ``abs_score`` = the largest scale * sum_d |q_d k_jd| of each row."""
    Hq, D = q.shape
    H, n = k.shape[0], k.shape[1]
    if n == 0:
        zero = np.zeros((Hq, D))
        return dict(out=zero, lse=np.full(Hq, -np.inf), weights=np.zeros((H, 0)), abs_out=zero, abs_score=np.zeros(Hq))
    g = q.reshape(H, Hq // H, D)
    s = np.einsum("hgd,hnd->hgn", g, k) * scale
    m = s.max(-1, keepdims=True)
    e = np.exp(s - m)
    total = e.sum(-1, keepdims=True)
    p = e / total
    return dict(
        out=np.einsum("hgn,hnd->hgd", p, v).reshape(Hq, D),
        lse=(m + np.log(total)).reshape(Hq),
        weights=p.sum(1),
        abs_out=np.einsum("hgn,hnd->hgd", p, np.abs(v)).reshape(Hq, D),
        abs_score=(np.einsum("hgd,hnd->hgn", np.abs(g), np.abs(k)) * abs(scale)).max(-1).reshape(Hq),
    )


def kept_positions(weights: np.ndarray, n: int, budget: int, recent: int) -> np.ndarray:
    """Positions of one (sequence, head) that an eviction keeps, in order."""
    if n <= budget:
        return np.arange(n)
    older = np.asarray(weights[: n - recent], dtype=np.float64)
    # stable sort of the negated weights: ties stay in order of position; NaN is above all
    order = np.argsort(np.where(np.isnan(older), -np.inf, -older), kind="stable")
    nan_first = np.concatenate([order[np.isnan(older[order])], order[~np.isnan(older[order])]])
    return np.sort(np.concatenate([nan_first[: budget - recent], np.arange(n - recent, n)]))


def token_scores(x: np.ndarray, token: int, top: int) -> dict[str, object]:
    """One row of logits (float64)."""
    V = x.shape[0]
    key = np.where(np.isnan(x), np.inf, x)
    order = np.lexsort((np.arange(V), -key, ~np.isnan(x)))[:top]
    m = x.max()
    if m == -np.inf:
        return dict(logprob=0.0 if token < 0 else -np.inf, entropy=0.0, ids=order, top=np.full(top, -np.inf))
    with np.errstate(invalid="ignore"):
        e = np.exp(x - m)
        total = e.sum()
        logp = x - m - np.log(total)
        p = e / total
        entropy = -np.where(p == 0, 0.0, p * np.where(p == 0, 0.0, logp)).sum()
    return dict(logprob=0.0 if token < 0 else logp[token], entropy=entropy, ids=order, top=logp[order])
