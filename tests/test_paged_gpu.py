"""The paged key-value cache on the GPU: append, decode and evict against
plain restatements (numpy, 64 bits), at the lengths, pages, layouts and masks
where they can go wrong.

Unused slots of every pool hold NaN, and unused page-table entries are out of
range, so a read past a sequence's end shows up in the results or in the device
status word.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
# relative error of rounding to a 16-bit format
ROUND = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


@pytest.fixture(autouse=True)
def healthy():
    from repercep_runtime_b200 import _lib

    _lib.device_status(reset=True)
    yield
    assert _lib.device_status(reset=True) == 0


def make_cache(pages, heads, page, D, kv, layout="bhsd"):
    """A pool whose every row is NaN (an e4m3 row: NaN bytes and scales)."""
    from repercep_runtime_b200 import paged

    cache = paged.alloc(pages, heads, page, D, DTYPES[kv], layout)
    for x in (cache.k, cache.v):
        if kv == "e4m3":
            x.view(torch.uint8).fill_(0x7F)
        else:
            x.fill_(float("nan"))
    for x in (cache.k_scales, cache.v_scales):
        if x is not None:
            x.fill_(float("nan"))
    return cache


def make_table(lengths, page, width=None, seed=0, first=0):
    """Shuffled pages; entries past a sequence's end are out of every range."""
    counts = [-(-n // page) for n in lengths]
    width = max(counts + [1]) if width is None else width
    ids = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(seed)) + first
    table = torch.full((len(lengths), width), 0x7FFFFFF0, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at : at + n].to(torch.int32)
        at += n
    return table.cuda(), sum(counts)


def heads_first(cache, x):
    x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
    return x if cache.layout == "bhsd" else x.transpose(1, 2)


def values(cache, name):
    """(pages, heads, page, D) float64 values of a pool."""
    x = getattr(cache, name)
    f = x.float() if cache.layout == "bhsd" else x.float().transpose(1, 2)
    f = f.double().cpu().numpy()
    scales = getattr(cache, name + "_scales")
    return f if scales is None else f * scales.double().cpu().numpy()[..., None]


def rows(shape, dtype, seed, factor=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * factor).to(dtype).cuda()


def filled(lengths, heads, page, D, kv, layout="bhsd", half=torch.bfloat16, seed=0, width=None, factor=1.0):
    """A cache with random rows at every position of every sequence."""
    from repercep_runtime_b200 import paged

    table, pages = make_table(lengths, page, width, seed)
    cache = make_cache(max(1, pages), heads, page, D, kv, layout)
    half = half if kv == "e4m3" else DTYPES[kv]
    n = sum(lengths)
    starts = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    zero = torch.zeros(len(lengths), dtype=torch.int32, device="cuda")
    k, v = rows((n, heads, D), half, seed + 1, factor), rows((n, heads, D), half, seed + 2, factor)
    got = paged.append(cache, k, v, table, zero, starts=starts)
    assert got.tolist() == lengths
    return cache, table, got, k, v


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
@pytest.mark.parametrize("kv, half", [("bf16", "bf16"), ("fp16", "fp16"), ("e4m3", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("D, page", [(32, 5), (64, 16), (128, 64), (256, 3)])
def test_append_writes_rows_and_nothing_else(kv, half, D, page, layout):
    from repercep_runtime_b200 import linear, paged

    H, before, new = 3, [0, 7, 16, 1], [4, 0, 1, 29]
    after = [a + b for a, b in zip(before, new)]
    table, pages = make_table(after, page, seed=3)
    cache = make_cache(pages, H, page, D, kv, layout)
    total = sum(new)
    # strided input, with rows that no sequence takes at both ends
    packed = rows((total + 3, H, 2, D), DTYPES[half], 5)
    packed[2, 0, 0, :4] = torch.tensor([1e4, -3e4, 0.0, 1.0]).to(DTYPES[half])
    packed[3, 1] = 0.0
    k, v = packed[:, :, 0], packed[:, :, 1]
    starts = (torch.tensor([0] + new).cumsum(0) + 1).to(torch.int32).cuda()
    lengths = torch.tensor(before, dtype=torch.int32).cuda()
    cap = table.shape[1] * page
    weights = torch.full((4, H, cap + 2), 7.0, device="cuda")
    got = paged.append(cache, k, v, table, lengths, starts=starts, weights=weights)
    assert got.tolist() == after and lengths.tolist() == before

    for name, x in (("k", k), ("v", v)):
        scale = None
        if kv == "e4m3":
            x8, scale = linear.quantize_rows(x.reshape(-1, D))
            x, scale = x8.contiguous().view(torch.uint8).view(-1, H, D), scale.view(-1, H)
        pool = heads_first(cache, getattr(cache, name))
        seen = torch.zeros(pool.shape[:3], dtype=torch.bool)
        at = 1
        for b, (n, add) in enumerate(zip(before, new)):
            for p in range(n, n + add):
                page_id, slot = int(table[b, p // page]), p % page
                assert torch.equal(pool[page_id, :, slot], x[at])
                if scale is not None:
                    assert torch.equal(getattr(cache, name + "_scales")[page_id, :, slot], scale[at])
                seen[page_id, :, slot] = True
                at += 1
        rest = pool[~seen.cuda()]
        assert bool((rest == 0x7F).all() if kv == "e4m3" else rest.isnan().all())
    for b, (n, add) in enumerate(zip(before, new)):
        assert bool((weights[b, :, n : n + add] == 0).all())
        assert bool((weights[b, :, :n] == 7).all()) and bool((weights[b, :, n + add :] == 7).all())


def test_append_one_token_each_and_non_finite_rows():
    from repercep_runtime_b200 import paged

    for kv in ("bf16", "e4m3"):
        table, pages = make_table([33, 1, 17], 16)
        cache = make_cache(pages, 2, 16, 64, kv)
        k, v = rows((3, 2, 64), torch.bfloat16, 1), rows((3, 2, 64), torch.bfloat16, 2)
        k[0, 0, 3], v[2, 1, 5] = float("nan"), float("inf")
        lengths = torch.tensor([32, 0, 16], dtype=torch.int32).cuda()
        assert paged.append(cache, k, v, table, lengths).tolist() == [33, 1, 17]
        got = values(cache, "k")[int(table[0, 2]), :, 0]
        assert np.isnan(got[0, 3]) and np.isfinite(got[1]).all()
        assert not np.isfinite(values(cache, "v")[int(table[2, 1]), 1, 0, 5])


# ------------------------------------------------------------------ decode
def check_decode(q, cache, table, lengths, weights=None, scale=None, got=None):
    """Runs decode and compares it with the 64-bit restatement.

    The bounds: with u the rounding of the 16-bit formats (the softmax weights'
    and the output's) and e = D 2^-23 max sum |q k| scale + 2^-20 a bound on a
    score's error in fp32 (products are exact, sums round once a term; exp and
    log of fp32 add a few 2^-22),
      |out - exact| <= u |exact| + (u + 2 e) sum_j p_j |v_j| + n 2^-23 max |v|
      |lse - exact| <= 2 e + 2^-21 |exact|,  |weight - exact| <= exact (4 e) + 2^-40
    (the third term of out: softmax weights below the 16-bit normal range)."""
    from repercep_runtime_b200 import paged

    scale64 = 1.0 / math.sqrt(cache.head_dim) if scale is None else scale
    before = None if weights is None else weights.double().cpu().numpy()
    out, lse = paged.decode(q, cache, table, lengths, scale=scale, weights=weights, return_lse=True, out=got)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    K, V = values(cache, "k"), values(cache, "v")
    tab = table.cpu().numpy()
    u = ROUND[q.dtype]
    u_p = ROUND[torch.bfloat16] if cache.dtype == torch.bfloat16 else ROUND[torch.float16]
    q64, out64, lse64 = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
    after = None if weights is None else weights.double().cpu().numpy()
    for b, n in enumerate(lengths.tolist()):
        k, v = op.gather_rows(K, tab[b], n), op.gather_rows(V, tab[b], n)
        ref = op.decode(q64[b], k, v, scale64)
        e = (cache.head_dim * 2.0**-23 * ref["abs_score"] + 2.0**-20)[:, None]
        tail = n * 2.0**-23 * (np.abs(v).max() if n else 0.0)
        bound = u * np.abs(ref["out"]) + (u_p + 2 * e) * ref["abs_out"] + tail
        assert (np.abs(out64[b] - ref["out"]) <= bound).all(), (b, n)
        if n == 0:
            assert (out64[b] == 0).all() and np.isneginf(lse64[b]).all()
        else:
            assert (np.abs(lse64[b] - ref["lse"]) <= 2 * e[:, 0] + 2.0**-21 * np.abs(ref["lse"])).all(), (b, n)
        if weights is not None:
            e_max = e.max()
            add = after[b, :, :n] - before[b, :, :n]
            slack = 2.0**-24 * np.maximum(np.abs(before[b, :, :n]), np.abs(after[b, :, :n]))
            assert (np.abs(add - ref["weights"]) <= 4 * e_max * ref["weights"] + slack + 2.0**-40).all(), (b, n)
            assert (after[b, :, n:] == before[b, :, n:]).all()
    return out, lse


LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 130, 300]


@pytest.mark.parametrize("layout, page", [("bhsd", 16), ("bshd", 64), ("bhsd", 7), ("bshd", 1)])
@pytest.mark.parametrize("kv, half", [("bf16", "bf16"), ("fp16", "fp16"), ("e4m3", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("D, H, G", [(128, 2, 1), (128, 1, 8), (64, 3, 5), (256, 2, 4), (32, 2, 16), (128, 1, 33)])
def test_decode_matches_the_definition(kv, half, D, H, G, layout, page):
    cache, table, lengths, _, _ = filled(LENGTHS, H, page, D, kv, layout, DTYPES[half], seed=D + G)
    q = rows((len(LENGTHS), H * G, D), DTYPES[half], 11, 2.0)
    weights = torch.rand((len(LENGTHS), H, table.shape[1] * page), generator=torch.Generator().manual_seed(4)).cuda()
    out, lse = check_decode(q, cache, table, lengths, weights)
    # without weights: the same bits
    from repercep_runtime_b200 import paged

    again = paged.decode(q, cache, table, lengths)
    assert torch.equal(again, out)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths", [[1], [513], [5000], [40000, 3, 0, 9999], [257] * 40])
def test_decode_splits_long_and_few_rows(kv, lengths):
    cache, table, n, _, _ = filled(lengths, 2, 32, 128, kv, seed=5)
    weights = torch.zeros((len(lengths), 2, table.shape[1] * 32), device="cuda")
    q = rows((len(lengths), 8, 128), torch.bfloat16, 12, 3.0)
    out, lse = check_decode(q, cache, table, n, weights)
    first = weights.clone()
    weights.zero_()
    again, lse2 = check_decode(q, cache, table, n, weights)
    assert torch.equal(out, again) and torch.equal(lse, lse2) and torch.equal(first, weights)


@pytest.mark.parametrize("kv", ["fp16", "e4m3"])
def test_decode_many_sequences(kv):
    """More sequences than a CTA has threads, many of them empty."""
    lengths = [(37 * i) % 211 if i % 3 else 0 for i in range(700)]
    cache, table, n, _, _ = filled(lengths, 1, 16, 64, kv, seed=6)
    q = rows((700, 4, 64), torch.float16 if kv == "fp16" else torch.bfloat16, 14)
    check_decode(q, cache, table, n, torch.zeros((700, 1, table.shape[1] * 16), device="cuda"))
    empty = torch.zeros_like(n)
    check_decode(q, cache, table, empty)


def test_decode_wide_table_strides_streams_and_scale():
    """A page table far wider than the sequences, q and out inside packed
    tensors, a table with padded rows, a scale of the caller's, another stream."""
    lengths = [100, 3, 77]
    cache, table, n, _, _ = filled(lengths, 2, 16, 128, "fp16", width=500, seed=9)
    wide = torch.full((3, 777), -5, dtype=torch.int32, device="cuda")
    wide[:, :500] = table
    packed = rows((3, 3, 4, 128), torch.float16, 13)
    out = torch.zeros((3, 6, 4, 128), dtype=torch.float16, device="cuda")[:, 2]
    check_decode(packed[:, 1], cache, wide[:, :500], n, torch.zeros((3, 2, 8003), device="cuda"), scale=0.3, got=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check_decode(packed[:, 1], cache, table, n, scale=0.02)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("kv", ["bf16", "fp16", "e4m3"])
def test_decode_extreme_scores(kv):
    """A few huge scores (the maximum moves late), values near the formats'
    ends, and rows of one repeated key."""
    from repercep_runtime_b200 import paged

    cache, table, n, k, v = filled([200, 64, 33], 1, 16, 128, kv, seed=21)
    q = rows((3, 4, 128), DTYPES["fp16" if kv == "fp16" else "bf16"], 22, 8.0)
    big = k.clone()
    big[150:160] *= 6.0
    big[200:264] = big[200]
    v2 = v * (100.0 if kv == "fp16" else 1e6)
    v2[10:20] *= 1e-6 if kv != "fp16" else 1e-4
    zero = torch.zeros_like(n)
    starts = torch.tensor([0, 200, 264, 297], dtype=torch.int32, device="cuda")
    paged.append(cache, big, v2, table, zero, starts=starts)
    check_decode(q, cache, table, n, torch.zeros((3, 1, table.shape[1] * 16), device="cuda"))


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_decode_passes_non_finite_rows_on(kv):
    """A NaN in a live key or value reaches its own sequence and head only."""
    from repercep_runtime_b200 import paged

    cache, table, n, k, v = filled([40, 40], 2, 16, 64, kv, seed=31)
    k2, v2 = k.clone(), v.clone()
    k2[3, 0, 1] = float("nan")
    v2[45, 1, 2] = float("inf")
    starts = torch.tensor([0, 40, 80], dtype=torch.int32, device="cuda")
    paged.append(cache, k2, v2, table, torch.zeros_like(n), starts=starts)
    q = rows((2, 4, 64), torch.bfloat16, 32)
    out, lse = paged.decode(q, cache, table, n, return_lse=True)
    assert bool(out[0, :2].isnan().all()) and bool(lse[0, :2].isnan().all())
    assert bool(out[0, 2:].isfinite().all()) and bool(out[1, :2].isfinite().all())
    assert not bool(out[1, 2:, 2].isfinite().any()) and bool(lse[1].isfinite().all())


def test_decode_shared_pages_and_offsets_past_32_bits():
    """Sequences that share their prefix pages, in a pool whose rows lie more
    than 2^31 elements apart."""
    from repercep_runtime_b200 import paged

    far = 1 << 30
    pools = [torch.empty(4 * far + 16 * 2 * 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k, v = (x.as_strided((5, 2, 16, 64), (far, 1024, 64, 1)) for x in pools)
    cache = paged.PagedKV(k, v)
    for i, x in enumerate((k, v)):
        x.copy_(rows((5, 2, 16, 64), torch.bfloat16, 41 + i))
    table = torch.tensor([[4, 1], [4, 3], [4, 0]], dtype=torch.int32, device="cuda")
    n = torch.tensor([20, 31, 16], dtype=torch.int32, device="cuda")
    check_decode(rows((3, 4, 64), torch.bfloat16, 43), cache, table, n, torch.zeros((3, 2, 32), device="cuda"))
    new = rows((3, 2, 64), torch.bfloat16, 44)
    got = paged.append(cache, new, new, table, torch.tensor([20, 31, 17], dtype=torch.int32, device="cuda"))
    assert got.tolist() == [21, 32, 18]
    assert torch.equal(k[3, :, 15], new[1]) and torch.equal(v[0, :, 1], new[2])


def test_decode_and_append_skip_what_does_not_fit_and_say_so():
    from repercep_runtime_b200 import _lib, paged

    cache, table, n, _, _ = filled([40, 40], 2, 16, 64, "bf16", seed=51)
    q = rows((2, 2, 64), torch.bfloat16, 52)
    good = paged.decode(q, cache, table, n)
    bad = table.clone()
    bad[0, 1] = 10**6
    out = paged.decode(q, cache, bad, n)
    assert _lib.device_status(reset=True) == 0x201
    assert torch.equal(out[1], good[1]) and bool(out.isfinite().all())
    out = paged.decode(q, cache, table, torch.tensor([-3, 40], dtype=torch.int32, device="cuda"))
    assert _lib.device_status(reset=True) == 0x202
    assert torch.equal(out[1], good[1]) and bool((out[0] == 0).all())
    before = cache.k.clone()
    new = rows((2, 2, 64), torch.bfloat16, 53)
    got = paged.append(cache, new, new, table, torch.tensor([48, 40], dtype=torch.int32, device="cuda"))
    assert _lib.device_status(reset=True) == 0x202 and got.tolist()[1] == 41
    cache.k[int(table[1, 2]), :, 8] = before[int(table[1, 2]), :, 8]
    assert torch.equal(cache.k.nan_to_num(), before.nan_to_num())


# ------------------------------------------------------------------- evict
def accumulated(shape, seed):
    """Weights over orders of magnitude, many of them equal."""
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn(shape, generator=g))
    w = torch.where(torch.rand(shape, generator=g) < 0.3, torch.zeros_like(w), w)
    w = torch.where(torch.rand(shape, generator=g) < 0.3, torch.full_like(w, 0.25), w)
    return w.cuda()


@pytest.mark.parametrize("layout, page", [("bhsd", 16), ("bshd", 5)])
@pytest.mark.parametrize("kv, D", [("bf16", 128), ("fp16", 32), ("e4m3", 64), ("e4m3", 256)])
@pytest.mark.parametrize("budget, recent", [(1, 0), (17, 17), (64, 0), (100, 33)])
def test_evict_keeps_the_heaviest_and_the_latest(kv, D, budget, recent, layout, page):
    from repercep_runtime_b200 import paged

    lengths, H = [0, 1, budget, budget + 1, 333, 65], 2
    kept_pages = [-(-min(n, budget) // page) for n in lengths]
    table, pages = make_table(lengths, page, seed=7)
    cache = make_cache(pages + sum(kept_pages), H, page, D, kv, layout)
    half = torch.bfloat16 if kv == "e4m3" else DTYPES[kv]
    total = sum(lengths)
    starts = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    paged.append(cache, rows((total, H, D), half, 8), rows((total, H, D), half, 9), table, torch.zeros_like(n), starts=starts)
    out_table, _ = make_table([min(x, budget) for x in lengths], page, -(-budget // page), seed=8, first=pages)
    w = accumulated((len(lengths), H, table.shape[1] * page + 3), 10)
    w[4, 0, 200], w[4, 1, 7] = float("nan"), float("inf")
    names = ["k", "v"] + (["k_scales", "v_scales"] if kv == "e4m3" else [])
    pools = {x: (heads_first(cache, getattr(cache, x)) if len(x) == 1 else getattr(cache, x)) for x in names}
    before = {x: p.cpu().clone() for x, p in pools.items()}
    got = paged.evict(cache, table, n, w, out_table, budget=budget, recent=recent)
    assert got.lengths.tolist() == [min(x, budget) for x in lengths] and n.tolist() == lengths
    after = {x: p.cpu() for x, p in pools.items()}
    kept, new_w, wc, tab, out_tab = (x.cpu() for x in (got.kept, got.weights, w, table, out_table))
    written = torch.zeros(before["k"].shape[:3], dtype=torch.bool)
    for b, length in enumerate(lengths):
        for h in range(H):
            want = op.kept_positions(wc[b, h].numpy(), length, budget, recent)
            assert kept[b, h, : len(want)].tolist() == want.tolist() and bool((kept[b, h, len(want) :] == -1).all())
            assert torch.equal(new_w[b, h, : len(want)].nan_to_num(), wc[b, h, want].nan_to_num())
            assert bool((new_w[b, h, len(want) :] == 0).all())
            for j, p in enumerate(want.tolist()):
                src, dst = (int(tab[b, p // page]), h, p % page), (int(out_tab[b, j // page]), h, j % page)
                for x in names:
                    assert torch.equal(after[x][dst], before[x][src])
                written[dst] = True
    for x in names:
        assert torch.equal(after[x][~written].nan_to_num(), before[x][~written].nan_to_num())


@pytest.mark.parametrize("n, budget, recent", [(5000, 4096, 100), (70000, 2048, 1024), (70000, 66000, 0), (20001, 1, 0)])
def test_evict_selects_exactly_in_long_sequences(n, budget, recent):
    from repercep_runtime_b200 import paged

    page, H = 128, 2
    table, pages = make_table([n], page)
    out_table, extra = make_table([min(n, budget)], page, first=pages)
    cache = paged.alloc(pages + extra, H, page, 32)
    w = accumulated((1, H, table.shape[1] * page), 12)
    w[0, 1] = torch.where(torch.rand(w.shape[2], generator=torch.Generator().manual_seed(1)).cuda() < 0.5, -w[0, 1], w[0, 1])
    got = paged.evict(cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), w, out_table, budget=budget, recent=recent)
    for h in range(H):
        assert got.kept[0, h].tolist() == op.kept_positions(w[0, h].cpu().numpy(), n, budget, recent).tolist()


@pytest.mark.parametrize("heads, width, n, budget", [(1, 6000, 750000, 5000), (256, 360, 3000, 700)])
def test_evict_without_room_for_the_keys_on_chip(heads, width, n, budget):
    """Page tables so wide that a CTA's slice of the weights does not fit shared
    memory: few rows (16 CTAs each) and many (one CTA each)."""
    from repercep_runtime_b200 import paged

    page = 128
    table, pages = make_table([n], page, width)
    out_table, extra = make_table([budget], page, first=pages)
    cache = paged.alloc(pages + extra, heads, page, 32, torch.float8_e4m3fn)
    w = accumulated((1, heads, width * page), 13)
    got = paged.evict(cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), w, out_table, budget=budget, recent=9)
    for h in range(0, heads, 51):
        assert got.kept[0, h].tolist() == op.kept_positions(w[0, h].cpu().numpy(), n, budget, 9).tolist()


# ---------------------------------------------------------------- refusals
def test_refusals():
    from repercep_runtime_b200 import _lib, paged

    cache, table, n, _, _ = filled([20, 3], 2, 16, 64, "bf16")
    q = rows((2, 4, 64), torch.bfloat16, 1)
    new = rows((2, 2, 64), torch.bfloat16, 2)
    w = torch.zeros((2, 2, 32), device="cuda")
    cases = [
        (lambda: paged.alloc(2, 2, 16, 96), "head dim"),
        (lambda: paged.PagedKV(cache.k, cache.v, layout="sbhd"), "layout"),
        (lambda: paged.PagedKV(cache.k, cache.v.half()), "k and v must both"),
        (lambda: paged.PagedKV(cache.k, cache.v[:1]), "one shape"),
        (lambda: paged.PagedKV(cache.k.to(torch.float8_e4m3fn), cache.v.to(torch.float8_e4m3fn)), "scales"),
        (lambda: paged.PagedKV(cache.k, cache.v.transpose(1, 2).contiguous().transpose(1, 2)), "strides"),
        (lambda: paged.decode(q[:, :3], cache, table, n), "multiple"),
        (lambda: paged.decode(q.half(), cache, table, n), "q must be"),
        (lambda: paged.decode(q[:1], cache, table, n), "q must be"),
        (lambda: paged.decode(q, cache, table.long(), n), "int32"),
        (lambda: paged.decode(q, cache, table, n[:1]), "lengths"),
        (lambda: paged.decode(q, cache, table, n, scale=-1.0), "scale"),
        (lambda: paged.decode(q, cache, table, n, scale=float("nan")), "scale"),
        (lambda: paged.decode(q, cache, table, n, weights=w[:, :, :31]), "positions"),
        (lambda: paged.decode(q, cache, table, n, weights=w[:, :1]), "weights"),
        (lambda: paged.decode(q, cache, table, n, weights=w[:1].expand(2, 2, 32)), "overlap"),
        (lambda: paged.decode(q.cpu(), cache, table, n), "q must be on"),
        (lambda: paged.append(cache, new[:1], new[:1], table, n), "starts"),
        (lambda: paged.append(cache, new[..., :32], new[..., :32], table, n), "k_new"),
        (lambda: paged.append(cache, new.half(), new.half(), table, n), "k_new"),
        (lambda: paged.append(cache, new, new, table, n, starts=n), "starts"),
        (lambda: paged.evict(cache, table, n, w, table, budget=0, recent=0), "budget"),
        (lambda: paged.evict(cache, table, n, w, table, budget=4, recent=5), "recent"),
        (lambda: paged.evict(cache, table, n, w, table[:, :1], budget=20, recent=5), "out_table"),
        (lambda: paged.evict(cache, table, n, w.half(), table, budget=4, recent=1), "weights"),
    ]
    for call, words in cases:
        with pytest.raises(ValueError, match=words):
            call()
    shifted = torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 4, 64)
    with pytest.raises(_lib.NativeError, match="RP_ERR_ALIGN"):
        paged.decode(shifted, cache, table, n)
    # nothing to do is no error
    empty = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert paged.decode(q[:0], cache, empty, none).shape == (0, 4, 64)
    assert paged.append(cache, new[:0], new[:0], empty, none).shape == (0,)
    assert paged.evict(cache, empty, none, torch.zeros((0, 2, 48), device="cuda"), empty, budget=4, recent=1).kept.shape == (0, 2, 4)
    flat = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    assert bool((paged.decode(q, cache, flat, torch.zeros_like(n)) == 0).all())


# --------------------------------------------------------------- other ways
def test_op_custom_op_and_graph_capture_agree():
    from repercep_runtime_b200 import ops, paged, scoring  # noqa: F401
    from repercep_runtime_b200.attention import PagedDecode

    cache, table, n, _, _ = filled([300, 7, 0, 65], 2, 16, 128, "e4m3", seed=61)
    q = rows((4, 8, 128), torch.bfloat16, 62)
    op = PagedDecode()
    assert op.available and op.supports(8, 2, 128) and not op.supports(8, 3, 128) and not op.supports(8, 2, 96)
    out, lse = op(q, cache, table, n, return_lse=True)
    got = torch.ops.repercep_b200.paged_decode(q, cache.k, cache.v, table, n, cache.k_scales, cache.v_scales)
    assert torch.equal(got[0], out) and torch.equal(got[1], lse)

    # append, decode with weights, evict and scores captured in one graph and replayed on new inputs
    weights = torch.zeros((4, 2, table.shape[1] * 16), device="cuda")
    wide, _ = make_table([301, 8, 1, 66], 16, table.shape[1] + 1, seed=61)
    pages = int(wide[wide < 1000].max()) + 1
    cut, extra = make_table([40, 8, 1, 40], 16, 3, first=pages)
    pool = make_cache(pages + extra, 2, 16, 128, "e4m3")
    lengths = torch.zeros(4, dtype=torch.int32, device="cuda")
    k, v = rows((372, 2, 128), torch.bfloat16, 63), rows((372, 2, 128), torch.bfloat16, 64)
    starts = torch.tensor([0, 300, 307, 307, 372], dtype=torch.int32, device="cuda")
    lengths = paged.append(pool, k, v, wide, lengths, starts=starts)
    weights = torch.zeros((4, 2, wide.shape[1] * 16), device="cuda")
    logits, tokens = rows((4, 5000), torch.bfloat16, 65), torch.tensor([1, 2, 3, 4999], device="cuda")
    new = rows((4, 2, 128), torch.bfloat16, 66)

    def step():
        after = paged.append(pool, new, new, wide, lengths, weights=weights)
        out, lse = paged.decode(q, pool, wide, after, weights=weights, return_lse=True)
        gone = paged.evict(pool, wide, after, weights, cut, budget=40, recent=8)
        return after, out, lse, *gone, *scoring.token_logprobs(logits, tokens, top=4)

    weights.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    q.copy_(rows((4, 8, 128), torch.bfloat16, 67))
    new.copy_(rows((4, 2, 128), torch.bfloat16, 68))
    logits.copy_(rows((4, 5000), torch.bfloat16, 69))
    weights.zero_()
    graph.replay()
    replayed = [t.clone() for t in captured]
    weights.zero_()
    for a, b in zip(replayed, step()):
        assert torch.equal(a, b)
    check_decode(q, pool, wide, captured[0])
