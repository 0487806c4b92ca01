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
            size = np.abs(vs)[:, None]
            floor = 2.0**-35 * (p * size).max(-1, keepdims=True) / np.where(size == 0.0, 1.0, size)
        else:
            floor = np.broadcast_to(2.0**-36 * p.max(-1, keepdims=True) if cache.dtype == torch.float16 else 0.0, p.shape)
        bound = op.decode_bound(q64[b], k, v, scale, u_out, u, floor.reshape(H * G, n))
        worst = np.abs(out64[b] - ref["out"]) / (bound["out"] + tiny + 1e-300)
        assert np.isfinite(out64[b]).all() and (worst <= 1).all(), (b, n, float(np.nanmax(worst)))
        assert (np.abs(lse64[b] - ref["lse"]) <= bound["lse"]).all(), (b, n)


@pytest.mark.parametrize("kv, half", [("bf16", "bf16"), ("fp16", "fp16"), ("e4m3", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("D, H, G", [(128, 2, 1), (64, 2, 8), (128, 1, 16), (256, 2, 4), (32, 1, 20)])
def test_what_is_rounded(kv, half, D, H, G):
    lengths = [1, 2, 3, 5, 6, 17, 64, 129, 300]
    cache, table, n, _, _ = filled(lengths, H, 16, D, kv, half=DTYPES[half], seed=D + G)
    check(rows((len(lengths), H * G, D), DTYPES[half], 5, 0.5), cache, table, n)


def one_far_key(n, at, D, log2_weight, half, seed):
    """q rows and keys of small scores, but for key ``at`` of each sequence,
    whose weight is about 2^log2_weight of the others'."""
    g = torch.Generator().manual_seed(seed)
    base = torch.randn((D,), generator=g).sign()
    q = (base + 0.05 * torch.randn((len(at), 4, D), generator=g)).to(half)
    k = 0.05 * torch.randn((len(at), n, 1, D), generator=g)
    for b, i in enumerate(at):
        k[b, i] = base * (log2_weight * math.log(2.0) / math.sqrt(D))
    return q.cuda(), k.to(half).cuda(), g


@pytest.mark.parametrize("half", ["bf16", "fp16"])
@pytest.mark.parametrize("ratio", [1e2, 1e4, 1e6, 1e7, 2.0**26, 1e12, 1e20])
def test_a_large_value_row_of_no_weight_costs_the_others_nothing(ratio, half):
    """e4m3: one V row ``ratio`` times the others, its key's weight 2^-100."""
    from repercep_runtime_b200 import paged

    if half == "fp16" and ratio > 1e6:
        pytest.skip("fp16 holds no such values")
    n, at, D = 520, [0, 100, 263, 519], 128
    q, k, g = one_far_key(n, at, D, -100.0, DTYPES[half], 3)
    small = 1e-2 if half == "fp16" else 1.0
    v = small * torch.randn((len(at), n, 1, D), generator=g)
    for b, i in enumerate(at):
        v[b, i] = (small * ratio * torch.randn((1, D), generator=g)).clamp(-6e4, 6e4) if half == "fp16" else (
            ratio * torch.randn((1, D), generator=g))
    cache, table, lengths, _, _ = filled([n] * len(at), 1, 16, D, "e4m3", half=DTYPES[half], seed=1)
    starts = torch.arange(0, len(at) * n + 1, n, dtype=torch.int32, device="cuda")
    paged.append(cache, k.view(-1, 1, D), v.to(DTYPES[half]).cuda().view(-1, 1, D), table, torch.zeros_like(lengths), starts=starts)
    check(q, cache, table, lengths)


@pytest.mark.parametrize("kv, half", [("bf16", "bf16"), ("fp16", "fp16"), ("e4m3", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("log2_weight", [4.0, 13.0, 20.0, 26.0, 30.0])
def test_small_weights_beside_a_dominant_key(kv, half, log2_weight):
    """A key 2^log2_weight times as heavy as each of the others, whose V row has
    nothing in most dimensions: the others make those."""
    from repercep_runtime_b200 import paged

    n, at, D = 1500, [0, 700, 1499], 64
    q, k, g = one_far_key(n, at, D, log2_weight, DTYPES[half], 4)
    v = 2e4 * (1.0 + 0.3 * torch.randn((len(at), n, 1, D), generator=g))
    for b, i in enumerate(at):
        v[b, i] = 0.0
        v[b, i, 0, :4] = 1.0
    cache, table, lengths, _, _ = filled([n] * len(at), 1, 32, D, kv, half=DTYPES[half], seed=2)
    starts = torch.arange(0, len(at) * n + 1, n, dtype=torch.int32, device="cuda")
    paged.append(cache, k.view(-1, 1, D), v.to(DTYPES[half]).cuda().view(-1, 1, D), table, torch.zeros_like(lengths), starts=starts)
    check(q, cache, table, lengths)


@pytest.mark.parametrize("kv, half", [("bf16", "bf16"), ("fp16", "fp16"), ("e4m3", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("ratio", [1e4, 1e8, 1e12, 1e25])
@pytest.mark.parametrize("steps", [(60.0,), (20.0, 40.0, 100.0), (-30.0, 5.5, 31.25)])
def test_large_value_rows_whose_weight_goes_later(kv, half, ratio, steps):
    """Keys of large V rows lead until later keys outweigh them by 2^60 and more:
    what those set must not hold the later ones down."""
    from repercep_runtime_b200 import paged

    if half == "fp16" and ratio > 1e8:
        pytest.skip("fp16 holds no such values")
    D, part, g = 64, 128 if len(steps) == 1 else 64, torch.Generator().manual_seed(8)
    n = part * (len(steps) + 1)
    base = torch.randn((D,), generator=g).sign()
    q = (base + 0.05 * torch.randn((3, 4, D), generator=g)).to(DTYPES[half]).cuda()
    level = torch.tensor([0.0, *steps]).repeat_interleave(part).view(1, n, 1, 1)  # log2 of the weights
    k = base * level * math.log(2.0) / math.sqrt(D) + 0.05 * torch.randn((3, n, 1, D), generator=g)
    top = 2e4 if half == "fp16" else ratio
    v = torch.randn((3, n, 1, D), generator=g) * torch.logspace(math.log10(top), math.log10(top / ratio), len(steps) + 1).repeat_interleave(part).view(1, n, 1, 1)
    cache, table, lengths, _, _ = filled([n] * 3, 1, 16, D, kv, half=DTYPES[half], seed=5)
    starts = torch.arange(0, 3 * n + 1, n, dtype=torch.int32, device="cuda")
    paged.append(cache, k.to(DTYPES[half]).cuda().view(-1, 1, D), v.clamp(-6e4, 6e4).to(DTYPES[half]).cuda().view(-1, 1, D) if half == "fp16"
                 else v.to(DTYPES[half]).cuda().view(-1, 1, D), table, torch.zeros_like(lengths), starts=starts)
    check(q, cache, table, lengths)


def test_negative_scales_of_large_rows():
    """A caller's own e4m3 cache may have multipliers of any sign."""
    cache, table, n, _, _ = filled([300, 40], 2, 16, 64, "e4m3", seed=4)
    cache.v_scales.copy_(torch.where(torch.arange(16, device="cuda") % 3 == 0, -1e6 * cache.v_scales, -cache.v_scales))
    cache.k_scales.neg_()
    check(rows((2, 4, 64), torch.bfloat16, 10), cache, table, n)


@pytest.mark.parametrize("kv", ["fp16", "e4m3"])
def test_scores_that_keep_rising(kv):
    """Ascending scores move the reference of the weights again and again; the
    V rows fall as they rise."""
    from repercep_runtime_b200 import paged

    n, D, half = 900, 64, torch.float16 if kv == "fp16" else torch.bfloat16
    g = torch.Generator().manual_seed(6)
    base = torch.randn((D,), generator=g).sign()
    q = base.repeat(1, 4, 1).to(half).cuda()
    k = (base * torch.linspace(0.0, 80.0, n).view(1, n, 1, 1) / math.sqrt(D)).to(half).cuda()
    v = (torch.randn((1, n, 1, D), generator=g) * torch.exp2(-torch.linspace(-8.0, 8.0, n)).view(1, n, 1, 1)).to(half).cuda()
    cache, table, lengths, _, _ = filled([n], 1, 16, D, kv, half=half, seed=3)
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    paged.append(cache, k.view(-1, 1, D), v.view(-1, 1, D), table, torch.zeros_like(lengths), starts=starts)
    check(q, cache, table, lengths)


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
