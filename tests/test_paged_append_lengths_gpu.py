"""Appends whose lengths or starts do not fit, on the GPU: what is written, what
is left alone, the lengths that come back and the device status."""

from __future__ import annotations

import pytest
import torch
from test_paged_gpu import DTYPES, filled, heads_first, rows

pytestmark = pytest.mark.gpu

BAD_LENGTH = 0x202


def status() -> int:
    from repercep_runtime_b200 import _lib

    return _lib.device_status(reset=True)


@pytest.fixture(autouse=True)
def healthy():
    status()
    yield
    assert status() == 0


def pools(cache):
    """The bytes of every tensor of a cache."""
    names = ("k", "v") + (("k_scales", "v_scales") if cache.k_scales is not None else ())
    return {x: getattr(cache, x).view(torch.uint8).clone() for x in names}


@pytest.mark.parametrize("kv, half", [("bf16", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("ragged", [False, True])
def test_a_negative_length_takes_no_token(kv, half, ragged):
    """Nothing of that sequence is written, and its length stays as it is: a
    length of 0 in its place would let the next call write over position 0."""
    from repercep_runtime_b200 import paged

    cache, table, n, _, _ = filled([20, 20, 20], 2, 16, 64, kv, half=DTYPES[half], seed=1)
    n[0], n[2] = -1, -2
    before = pools(cache)
    counts = [2, 3, 1] if ragged else [1, 1, 1]
    starts = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda() if ragged else None
    new = rows((sum(counts), 2, 64), DTYPES[half], 2)
    weights = torch.full((3, 2, table.shape[1] * 16), 7.0, device="cuda")
    got = paged.append(cache, new, new, table, n, starts=starts, weights=weights)
    assert status() == BAD_LENGTH
    assert got.tolist() == [-1, 20 + counts[1], -2]
    assert bool((weights[[0, 2]] == 7).all())
    after = pools(cache)
    page = int(table[1, 1])  # where sequence 1 took its tokens, from slot 4 on
    for name, x in after.items():
        unit = 4 if "scales" in name else 1  # bytes of a scale lie in the slots' dimension
        taken = (page, slice(None), slice(4 * unit, (4 + counts[1]) * unit))
        assert not torch.equal(x[taken], before[name][taken])
        x[taken] = before[name][taken]
        assert torch.equal(x, before[name]), name


@pytest.mark.parametrize("kv", ["fp16", "e4m3"])
def test_lengths_stop_at_the_end_of_the_table(kv):
    """Tokens that fit are stored, and the lengths count these alone, so that
    the calls after it have lengths that fit."""
    from repercep_runtime_b200 import paged

    cache, table, n, _, _ = filled([48, 48, 48, 48, 48], 1, 16, 64, kv, half=torch.float16, seed=3)
    n = torch.tensor([46, 48, 60, 10, 2**31 - 2], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 3, 6, 9, 12, 15], dtype=torch.int32, device="cuda")
    new = rows((15, 1, 64), torch.float16, 4)
    before = pools(cache)
    got = paged.append(cache, new, new, table, n, starts=starts)
    assert status() == BAD_LENGTH
    assert got.tolist() == [48, 48, 48, 13, 48]
    changed = torch.zeros((cache.num_pages, 16), dtype=torch.bool, device="cuda")
    for b, p in [(0, 46), (0, 47), (3, 10), (3, 11), (3, 12)]:
        changed[table[b, p // 16].long(), p % 16] = True
    differs = (heads_first(cache, cache.k).contiguous().view(torch.uint8) != before["k"].view(cache.num_pages, 1, 16, -1)).any(-1)[:, 0]
    assert torch.equal(differs, changed)
    paged.decode(rows((5, 1, 64), torch.float16, 5), cache, table, got)
    assert status() == 0
    # one token each
    got = paged.append(cache, new[:5], new[:5], table, torch.tensor([47, 48, 49, 0, 2**31 - 1], dtype=torch.int32, device="cuda"))
    assert status() == BAD_LENGTH and got.tolist() == [48, 48, 48, 1, 48]


def test_starts_outside_the_new_tokens_count_what_is_there():
    """Lengths grow by the tokens that were given, and a sequence's first one
    goes right behind its length."""
    from repercep_runtime_b200 import paged

    new = rows((4, 2, 64), torch.bfloat16, 6)
    for starts, counts, first in [([0, 2, 9], [2, 2], [0, 2]), ([-3, 2, 4], [2, 2], [0, 2]), ([0, 7, 9], [4, 0], [0, 4])]:
        cache, table, n, _, _ = filled([20, 25], 2, 16, 64, "bf16", width=2, seed=7)
        got = paged.append(cache, new, new, table, n, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
        assert status() == BAD_LENGTH, starts
        assert got.tolist() == [20 + counts[0], 25 + counts[1]], starts
        for b, (length, count, at) in enumerate(zip((20, 25), counts, first)):
            for i in range(count):
                p = length + i
                assert torch.equal(cache.k[int(table[b, p // 16]), :, p % 16], new[at + i]), (starts, b, i)


def test_descending_starts_are_reported():
    from repercep_runtime_b200 import paged

    cache, table, n, _, _ = filled([3, 4, 5], 2, 16, 64, "bf16", seed=8)
    new = rows((6, 2, 64), torch.bfloat16, 9)
    got = paged.append(cache, new, new, table, n, starts=torch.tensor([0, 4, 2, 6], dtype=torch.int32, device="cuda"))
    assert status() == BAD_LENGTH and got.tolist()[1] == 4
