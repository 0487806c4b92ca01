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


def decode_bound(
    q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float, out_round: float, weight_round: float, floor: np.ndarray
) -> dict[str, np.ndarray]:
    """Bounds on the rounding errors of one sequence's decode, element by element.

    Scores are fp32 sums of exact products: e_j = D 2^-23 scale sum_d |q_d k_jd|
    + 2^-20 bounds key j's (the constant also takes exp and log in fp32), and
    e = sum_j p_j e_j the log-sum-exp's.  The sums over keys take fp32 steps of
    16 keys in 4 or more chains, two products a step: n / 32 + 8 steps, each off
    by 2^-21 of what it adds to.  A weight is rounded by ``weight_round`` of
    itself, or by ``floor`` (Hq, n) in units of the exact weights where that is
    more; the output once by ``out_round``.

    ``out`` (Hq, D), ``lse`` (Hq,)."""
    ref = decode(q, k, v, scale)
    Hq, D = q.shape
    H, n = k.shape[0], k.shape[1]
    if n == 0:
        return dict(out=np.zeros((Hq, D)), lse=np.zeros(Hq))
    g = q.reshape(H, Hq // H, D)
    s = np.einsum("hgd,hnd->hgn", g, k) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    e = D * 2.0**-23 * abs(scale) * np.einsum("hgd,hnd->hgn", np.abs(g), np.abs(k)) + 2.0**-20
    e_lse = (p * e).sum(-1)
    chain = (n / 32 + 8) * 2.0**-21
    each = p * (weight_round + 2 * e + 2 * e_lse[..., None] + 2 * chain) + floor.reshape(H, Hq // H, n)
    out = np.einsum("hgn,hnd->hgd", each, np.abs(v)).reshape(Hq, D) * (1 + out_round)
    return dict(out=out + out_round * np.abs(ref["out"]), lse=2 * e_lse.reshape(Hq) + chain + 2.0**-21 * np.abs(ref["lse"]))
