"""Decode under element-wise bounds (``oracle.paged.decode_bound``): what it
rounds at ordinary values, and weights and V rows of very different size.

The bounds of a softmax weight: two 16-bit parts are off by the square of the
format's rounding; an e4m3 cache's one fp16 value, which carries the V scale
too, by 2^-11.  fp16 values are held to 2^-25 absolutely, in units in which the
largest weight (e4m3: the largest product of weight and V scale) is at least
2^11 (2^10): the floors below.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch
from test_paged_gpu import DTYPES, ROUND, filled, rows

from oracle import paged as op

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def healthy():
    from repercep_runtime_b200 import _lib

    _lib.device_status(reset=True)
    yield
    assert _lib.device_status(reset=True) == 0


def dequantized(cache, name):
    """(pages, heads, page, D) float64 values and (pages, heads, page) scales; a
    row whose scale is 0 is zeros."""
    x = getattr(cache, name)
    f = x.float().double().cpu().numpy()
    f = f if cache.layout == "bhsd" else f.swapaxes(1, 2)
    scales = getattr(cache, name + "_scales")
    if scales is None:
        return f, np.ones(f.shape[:3])
    s = scales.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        return np.where(s[..., None] == 0.0, 0.0, f * s[..., None]), s


def check(q, cache, table, lengths):
    from repercep_runtime_b200 import paged

    out, lse = paged.decode(q, cache, table, lengths, return_lse=True)
    D, scale = cache.head_dim, 1.0 / math.sqrt(cache.head_dim)
    (K, _), (V, V_scales) = dequantized(cache, "k"), dequantized(cache, "v")
    e4m3 = cache.k_scales is not None
    u_out, u = ROUND[q.dtype], 2.0**-11 if e4m3 else ROUND[cache.dtype] ** 2
    tiny = 2.0**-25 if q.dtype == torch.float16 else 0.0  # an output below fp16's normal range
    q64, out64, lse64 = (t.double().cpu().numpy() for t in (q, out, lse))
    for b, n in enumerate(lengths.tolist()):
        row = table[b].cpu().numpy()
        k, v, vs = (op.gather_rows(x, row, n) for x in (K, V, V_scales))
        ref = op.decode(q64[b], k, v, scale)
        H, G = k.shape[0], q.shape[1] // k.shape[0]
        s = np.einsum("hgd,hnd->hgn", q64[b].reshape(H, G, D), k) * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        if e4m3:
            safe = np.where(vs == 0.0, 1.0, vs)[:, None]
            floor = 2.0**-35 * (p * vs[:, None]).max(-1, keepdims=True) / safe
        else:
            floor = np.broadcast_to(2.0**-36 * p.max(-1, keepdims=True) if cache.dtype == torch.float16 else 0.0, p.shape)
        bound = op.decode_bound(q64[b], k, v, scale, u_out, u, floor.reshape(H * G, n))
        worst = np.abs(out64[b] - ref["out"]) / (bound["out"] + tiny + 1e-300)
        assert np.isfinite(out64[b]).all() and (worst <= 1).all(), (b, n, float(np.nanmax(worst)))
        assert (np.abs(lse64[b] - ref["lse"]) <= bound["lse"]).all(), (b, n)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
def test_zero_and_tiny_fp16_rows_in_an_e4m3_cache(D, layout):
    """The scale of an fp16 row below 1.27e-5 rounds to 0: such a row is zeros,
    in its own sequence and in the sums of the others."""
    from repercep_runtime_b200 import paged

    lengths = [1, 16, 70, 200]
    cache, table, n, k, v = filled(lengths, 2, 16, D, "e4m3", layout, torch.float16, seed=D)
    at = [0, 1, 1 + 5, 17, 17 + 33, 17 + 69, 87, 87 + 64, 87 + 199]
    for i in at:  # zeros, and tiny values among zeros
        k[i, 0], v[i, 1] = 0.0, 0.0
        k[i, 1], v[i, 0] = 0.0, 0.0
        k[i, 1, ::3], v[i, 0, 1::2] = 1e-5, -1.2e-5
    starts = torch.tensor([0, 1, 17, 87, 287], dtype=torch.int32, device="cuda")
    paged.append(cache, k, v, table, torch.zeros_like(n), starts=starts)
    q = rows((4, 8, D), torch.float16, 9)
    check(q, cache, table, n)
    # against the rows that went in: an e4m3 value is within 2^-4 of itself (or of its row's
    # amax 2^-9), so a score within 2^-4 sum |q k| and a weight's share within twice that
    out = paged.decode(q, cache, table, n).double().cpu().numpy()
    pages = [x.double().cpu().numpy().swapaxes(0, 1) for x in (k, v)]
    for b, (s, e) in enumerate(zip([0, 1, 17, 87], [1, 17, 87, 287])):
        ref = op.decode(q[b].double().cpu().numpy(), pages[0][:, s:e], pages[1][:, s:e], D**-0.5)
        share = 2.0**-4 + 2 * 2.0**-4 * ref["abs_score"][:, None]
        assert (np.abs(out[b] - ref["out"]) <= (share + 2.0**-8) * ref["abs_out"] + 2.0**-8).all(), b
    # moved by an eviction, they stay what they were
    free = torch.arange(cache.num_pages, cache.num_pages + 4, dtype=torch.int32, device="cuda").view(1, 4)
    pool = paged.PagedKV(*(torch.cat([x, torch.zeros_like(x[:4])]) if x.dtype != paged.FP8 else
                           torch.cat([x.view(torch.uint8), torch.zeros_like(x[:4].view(torch.uint8))]).view(paged.FP8)
                           for x in (cache.k, cache.v, cache.k_scales, cache.v_scales)), layout)
    weights = torch.zeros((1, 2, table.shape[1] * 16), device="cuda")
    weights[:, :, 64] = 1.0
    got = paged.evict(pool, table[3:4], n[3:4], weights, free, budget=64, recent=40)
    assert bool((got.kept == 64).any())
    check(q[3:4], pool, free, got.lengths)
