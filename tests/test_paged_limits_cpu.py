"""Limits of the paged decode's arguments that the C ABI checks, without a GPU."""

from __future__ import annotations

import pytest
from test_paged_cpu import decode, lib  # noqa: F401


@pytest.mark.parametrize("scale", [3e38, -3e38, float("inf")])
def test_a_scale_that_log2_units_do_not_hold_is_refused(lib, scale):  # noqa: F811
    assert decode(lib, scale=scale) == -1 and b"finite" in lib.rp_last_error()
