"""Paged decode attention as an op, beside the shared-prefix candidate decode.

``SharedPrefixFP8Decode`` reads one fixed prefix and a fresh suffix;
``PagedDecode`` is one new token per sequence over a cache that grows: the
token-VLA decode of the reference (``VLAEngine.plan``, src/repercep/models/
vla.py:229-258) on ``repercep_runtime_b200.paged``, with grouped query heads.
"""

from __future__ import annotations

from typing import TYPE_CHECKING

from repercep_runtime_b200.attention.fp8_b200 import b200_device_present

if TYPE_CHECKING:
    import torch

    from repercep_runtime_b200.paged import PagedKV


class PagedDecode:
    """Attention of one new token per sequence over a paged key-value cache."""

    name = "b200-paged-decode"

    def __init__(self) -> None:
        self._import_error: str | None = None
        try:
            from repercep_runtime_b200 import _lib

            _lib.load()
        except Exception as e:
            self._import_error = f"{type(e).__name__}: {e}"
        if self._import_error is None and not b200_device_present():
            self._import_error = "no sm_100 (B200) CUDA device visible"

    @property
    def available(self) -> bool:
        return self._import_error is None

    def supports(self, heads: int, kv_heads: int, head_dim: int) -> bool:
        from repercep_runtime_b200 import paged

        return (
            self.available
            and head_dim in paged.HEAD_DIMS
            and 1 <= kv_heads <= 65535
            and 1 <= heads <= 65535
            and heads % kv_heads == 0
        )

    def __call__(
        self,
        query: torch.Tensor,
        cache: PagedKV,
        page_table: torch.Tensor,
        lengths: torch.Tensor,
        *,
        scale: float | None = None,
        weights: torch.Tensor | None = None,
        out: torch.Tensor | None = None,
        return_lse: bool = False,
    ):  # type: ignore[no-untyped-def]
        if self._import_error is not None:
            raise RuntimeError(f"B200 paged decode is not available ({self._import_error})")
        from repercep_runtime_b200 import paged

        return paged.decode(
            query, cache, page_table, lengths, scale=scale, weights=weights, out=out, return_lse=return_lse
        )


__all__ = ["PagedDecode"]
