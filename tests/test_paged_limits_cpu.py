"""Limits of the paged decode's arguments that the C ABI checks, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
from test_paged_cpu import DUMMY, append, decode, evict, kv, lib  # noqa: F401


@pytest.mark.parametrize("scale", [3e38, -3e38, float("inf")])
def test_a_scale_that_log2_units_do_not_hold_is_refused(lib, scale):  # noqa: F811
    assert decode(lib, scale=scale) == -1 and b"finite" in lib.rp_last_error()


def test_tables_whose_loops_would_pass_2_31_are_refused(lib):  # noqa: F811
    """A loop over positions steps past its end by up to 2^23: an int that wraps
    there would index memory before the weights."""
    pages = (2**31 - 8192) // 16
    n = ctypes.c_size_t()
    assert lib.rp_paged_decode_workspace_bytes(kv(), 1, 2, pages, 1, ctypes.byref(n)) == -2
    assert b"2^31" in lib.rp_last_error()
    for call in (append, decode, evict):
        assert call(lib, pages=pages, stride=pages, weights=DUMMY, cols=1 << 31) == -2 and b"2^31" in lib.rp_last_error()
    assert lib.rp_paged_decode_workspace_bytes(kv(), 1, 2, (2**31 - 2**24) // 16, 1, ctypes.byref(n)) == 0


def test_more_query_rows_than_an_int_holds_are_refused(lib):  # noqa: F811
    """B * query heads numbers the items that CTAs leave to each other."""
    assert decode(lib, B=65535, Hq=40000) == -2 and b"2^31" in lib.rp_last_error()


def test_a_stride_that_no_offset_uses_is_any_number(lib):  # noqa: F811
    """One sequence, one page, one head: the call gets as far as the workspace."""
    for pool, changes in [(None, dict(B=1, q_strides=(513, 128))), (kv(num_pages=1, strides=(4097, 2048, 128)), {}),
                          (kv(heads=1, strides=(2048, 3, 128)), {}), (kv(page_size=1, strides=(256, 128, 5)), {})]:
        assert decode(lib, pool, ws=None, **changes) == -6, lib.rp_last_error()
