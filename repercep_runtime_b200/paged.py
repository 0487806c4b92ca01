"""Paged key-value cache of a token-VLA decode on B200 (librepercep_b200.so).

The reference decodes its action candidates through HF ``generate``, whose
cache holds every candidate's prompt again (scripts/run_vla_openvla_gpu.py:
174-186; ``VLAEngine.plan``, src/repercep/models/vla.py:229-258).  Here a cache
is one pool of pages that sequences take as they grow and may share:

  append  new tokens' K and V rows into the pages (quantized on the way into
          an e4m3 cache, one scale per row);
  decode  attention of one new token per sequence over its cached tokens, with
          grouped query heads; on request every key's attention weight is
          added to the sequence's accumulated weights;
  evict   every sequence cut to a budget of tokens per KV head, the recent ones
          and those of the greatest accumulated weight, into other pages.

Position p of sequence b is slot ``p % page_size`` of page ``page_table[b, p //
page_size]``.  Tables and lengths are int32 CUDA tensors and stay on the device
(no call synchronises); entries past a sequence's pages are not read.  What
does not fit is recorded in the device's status word (``_lib.device_status``):
a row whose page id is outside the pool and a new token past the page table are
skipped, a length is read as the nearest valid one, and a sequence of negative
length takes no new token.

Torch allocates outputs and workspaces and supplies the current stream; the
arithmetic runs in the library, which has no fallback (a missing library
raises).
"""

from __future__ import annotations

import functools
from ctypes import byref, c_float, c_int64
from dataclasses import dataclass, field
from typing import NamedTuple

import torch

from . import _lib

FP8 = torch.float8_e4m3fn
HEAD_DIMS = (32, 64, 128, 256)
_HALF = {torch.bfloat16: _lib.RP_DTYPE_BF16, torch.float16: _lib.RP_DTYPE_F16}
_KV = {torch.bfloat16: _lib.RP_KV_BF16, torch.float16: _lib.RP_KV_F16, FP8: _lib.RP_KV_E4M3}
_I64x2 = c_int64 * 2
_I64x4 = c_int64 * 4


@dataclass(frozen=True, eq=False)
class PagedKV:
    """A pool of pages: ``k`` and ``v`` (pages, heads, page_size, D) for layout
    "bhsd" (a page in the place of a batch), (pages, page_size, heads, D) for
    "bshd"; bf16, fp16, or e4m3 with fp32 ``k_scales`` / ``v_scales`` (pages,
    heads, page_size), one dequant multiplier per row; a row whose scale is 0 is
    zeros, whatever its bytes (``append`` leaves such a row for fp16 values all
    below 1.27e-5).  D is unit-stride and k and v share their strides."""

    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor | None = None
    v_scales: torch.Tensor | None = None
    layout: str = "bhsd"
    num_pages: int = field(init=False)
    heads: int = field(init=False)
    page_size: int = field(init=False)
    head_dim: int = field(init=False)
    dtype: torch.dtype = field(init=False)
    device: torch.device = field(init=False)

    def __post_init__(self) -> None:
        k, v = self.k, self.v
        if self.layout not in ("bhsd", "bshd"):
            raise ValueError(f"unknown layout {self.layout!r}")
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError("k and v must be 4-D of one shape")
        if k.dtype != v.dtype or k.dtype not in _KV:
            raise ValueError(f"k and v must both be bf16, fp16 or float8_e4m3fn, got {k.dtype} and {v.dtype}")
        if not k.is_cuda or k.device != v.device:
            raise ValueError("k and v must be CUDA tensors on one device")
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("k and v must share their strides, with a unit-stride head dim")
        bhsd = self.layout == "bhsd"
        pages, heads, size, D = k.shape if bhsd else (k.shape[0], k.shape[2], k.shape[1], k.shape[3])
        if D not in HEAD_DIMS:
            raise ValueError(f"head dim {D} not in {HEAD_DIMS}")
        for name, scales in (("k_scales", self.k_scales), ("v_scales", self.v_scales)):
            if (scales is None) != (k.dtype != FP8):
                raise ValueError(f"{name}: an e4m3 cache has scales, a 16-bit one has none")
            if scales is not None and (
                tuple(scales.shape) != (pages, heads, size)
                or scales.dtype != torch.float32
                or scales.device != k.device
                or not scales.is_contiguous()
            ):
                raise ValueError(f"{name} must be contiguous fp32 ({pages}, {heads}, {size}) on {k.device}")
        for name, value in (("num_pages", pages), ("heads", heads), ("page_size", size), ("head_dim", D)):
            object.__setattr__(self, name, int(value))
        object.__setattr__(self, "dtype", k.dtype)
        object.__setattr__(self, "device", k.device)
        s = k.stride()
        strides = s[:3] if bhsd else (s[0], s[2], s[1])
        object.__setattr__(self, "_geometry", (strides, _KV[k.dtype], self.num_pages, self.heads, self.page_size, D))
        object.__setattr__(self, "_kv", _lib.PagedKVStruct(*self._pointers(), *self._geometry))

    def _pointers(self) -> tuple[int | None, ...]:
        ks, vs = self.k_scales, self.v_scales
        return (
            self.k.data_ptr(), self.v.data_ptr(),
            None if ks is None else ks.data_ptr(), None if vs is None else vs.data_ptr(),
        )  # fmt: skip

    def _struct(self):  # type: ignore[no-untyped-def]
        """A pointer to ``rp_paged_kv`` of the tensors as they are now."""
        kv, now = self._kv, self._pointers()
        if (kv.k, kv.v, kv.k_scales, kv.v_scales) != now:  # a tensor was given another storage
            kv = _lib.PagedKVStruct(*now, *self._geometry)
        return byref(kv)


def alloc(
    num_pages: int,
    heads: int,
    page_size: int,
    head_dim: int,
    dtype: torch.dtype = torch.bfloat16,
    layout: str = "bhsd",
    device: torch.device | str = "cuda",
) -> PagedKV:
    """A zeroed pool of ``num_pages`` pages."""
    shape = (num_pages, heads, page_size, head_dim) if layout == "bhsd" else (num_pages, page_size, heads, head_dim)
    k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    scales: list[torch.Tensor | None] = [None, None]
    if dtype == FP8:
        scales = [torch.zeros((num_pages, heads, page_size), dtype=torch.float32, device=device) for _ in range(2)]
    return PagedKV(k, v, scales[0], scales[1], layout)


def _int32(x: torch.Tensor, name: str, shape: tuple[int, ...], device: torch.device) -> None:
    if x.dtype != torch.int32 or x.device != device or x.shape != shape:
        raise ValueError(f"{name} must be int32 {shape} on {device}, got {x.dtype} {tuple(x.shape)} on {x.device}")


def _table(device: torch.device, name: str, table: torch.Tensor, B: int | None = None) -> tuple[int, int, int]:
    """Checks a page table; (sequences, pages a row, row stride)."""
    if table.dim() != 2:
        raise ValueError(f"{name} must be 2-D (sequences, pages)")
    rows, pages = table.shape
    _int32(table, name, (rows if B is None else B, pages), device)
    stride, step = table.stride()
    if pages > 1 and step != 1:
        raise ValueError(f"{name} rows must be contiguous")
    return rows, pages, stride if rows > 1 else pages


def _lengths(device: torch.device, lengths: torch.Tensor, B: int) -> None:
    _int32(lengths, "lengths", (B,), device)
    if B > 1 and lengths.stride(0) != 1:
        raise ValueError("lengths must be contiguous")


def _weights(cache: PagedKV, w: torch.Tensor | None, B: int, pages: int):  # type: ignore[no-untyped-def]
    """(pointer, strides, columns) of accumulated weights."""
    if w is None:
        return None, None, 0
    if w.dim() != 3 or w.dtype != torch.float32 or w.device != cache.device:
        raise ValueError(f"weights must be fp32 ({B}, {cache.heads}, positions) on {cache.device}")
    rows, heads, cols = w.shape
    if rows != B or heads != cache.heads:
        raise ValueError(f"weights must be fp32 ({B}, {cache.heads}, positions) on {cache.device}")
    if cols < pages * cache.page_size:
        raise ValueError(f"weights hold {cols} positions, the page table {pages * cache.page_size}")
    s0, s1, s2 = w.stride()
    if cols > 1 and s2 != 1:
        raise ValueError("weights must have unit-stride positions")
    if (B > 1 and s0 == 0) or (heads > 1 and s1 == 0):
        raise ValueError("weights of sequences or heads overlap")
    return w.data_ptr(), _I64x2(s0, s1), cols


def append(
    cache: PagedKV,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    starts: torch.Tensor | None = None,
    weights: torch.Tensor | None = None,
) -> torch.Tensor:
    """Writes new tokens' rows ``k_new`` / ``v_new`` (tokens, heads, D), bf16 or
    fp16, behind the sequences' ``lengths``; returns the lengths after it.

    ``starts`` (sequences + 1,) int32 holds the first new token of each
    sequence (tokens outside [starts[0], starts[-1]) are left out, starts outside
    the new tokens count as their ends); without it
    every sequence gets one token.  An e4m3 cache takes each row's scale and
    bytes from ``linear.quantize_rows``'s recipe.  ``weights`` are zeroed at
    the new positions.  Tokens past the page table are not counted; a sequence
    of negative length takes nothing and keeps that length."""
    device, dtype = cache.device, k_new.dtype
    B, pages, row = _table(device, "page_table", page_table)
    _lengths(device, lengths, B)
    if k_new.dim() != 3 or k_new.shape != v_new.shape or k_new.shape[1:] != (cache.heads, cache.head_dim):
        raise ValueError(f"k_new and v_new must be (tokens, {cache.heads}, {cache.head_dim})")
    if dtype not in _HALF or v_new.dtype != dtype or (cache.dtype != FP8 and dtype != cache.dtype):
        raise ValueError(f"k_new and v_new must be {'bf16 or fp16' if cache.dtype == FP8 else cache.dtype}, got {dtype}")
    if k_new.device != device or v_new.device != device:
        raise ValueError(f"k_new and v_new must be on {device}")
    (k0, k1, k2), (v0, v1, v2) = k_new.stride(), v_new.stride()
    if k2 != 1 or v2 != 1:
        raise ValueError("k_new and v_new must have a unit-stride head dim")
    tokens = k_new.shape[0]
    if starts is not None:
        _int32(starts, "starts", (B + 1,), device)
        if starts.stride(0) != 1:
            raise ValueError("starts must be contiguous")
    elif tokens != B:
        raise ValueError(f"{tokens} new tokens for {B} sequences need starts")
    w, w_strides, w_cols = _weights(cache, weights, B, pages)
    out = torch.empty_like(lengths)
    _lib.launch(
        device.index, "rp_paged_append", cache._struct(), k_new.data_ptr(), v_new.data_ptr(),
        _I64x4(k0, k1, v0, v1), _HALF[dtype], tokens, None if starts is None else starts.data_ptr(),
        page_table.data_ptr(), row, pages, lengths.data_ptr(), B, w, w_strides, w_cols, out.data_ptr(),
    )  # fmt: skip
    return out


@functools.lru_cache(maxsize=1024)
def _decode_workspace(geometry: tuple, B: int, Hq: int, pages: int, with_weights: bool) -> int:
    """``rp_paged_decode_workspace_bytes`` of a pool's geometry."""
    need = _lib._c_size_t(0)
    kv = _lib.PagedKVStruct(None, None, None, None, *geometry)
    rc = _lib.load().rp_paged_decode_workspace_bytes(byref(kv), B, Hq, pages, int(with_weights), byref(need))
    _lib.check("rp_paged_decode_workspace_bytes", rc)
    return int(need.value)


def decode(
    q: torch.Tensor,
    cache: PagedKV,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: float | None = None,
    weights: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
):  # type: ignore[no-untyped-def]
    """Attention of one query token per sequence, ``q`` (sequences, query heads,
    D), over the ``lengths`` cached tokens of each (the new token's own row
    among them, if it was appended before).  Query heads share KV heads in
    groups (query heads a multiple of ``cache.heads``).

    Returns ``out`` in q's shape and type, and with ``return_lse`` the fp32
    natural log-sum-exp (sequences, query heads).  A sequence of length 0 gives
    zeros and -inf.  ``weights`` fp32 (sequences, heads, positions): every
    key's attention weight, summed over the query heads of its KV head, is
    added in place."""
    device, dtype = cache.device, q.dtype
    B, pages, row = _table(device, "page_table", page_table)
    _lengths(device, lengths, B)
    shape = q.shape
    if len(shape) != 3 or shape[0] != B or shape[2] != cache.head_dim:
        raise ValueError(f"q must be ({B}, query heads, {cache.head_dim}), got {tuple(shape)}")
    Hq = shape[1]
    if Hq == 0 or Hq % cache.heads != 0:
        raise ValueError(f"{Hq} query heads are no multiple of {cache.heads} KV heads")
    if dtype not in _HALF or (cache.dtype != FP8 and dtype != cache.dtype):
        raise ValueError(f"q must be {'bf16 or fp16' if cache.dtype == FP8 else cache.dtype}, got {dtype}")
    if q.device != device:
        raise ValueError(f"q must be on {device}")
    q0, q1, q2 = q.stride()
    if q2 != 1:
        raise ValueError("q must have a unit-stride head dim")
    if scale is not None:
        given, scale = scale, c_float(scale).value  # as the library takes it, where 0 means 1 / sqrt(D)
        if not 0.0 < scale < float("inf"):
            raise ValueError(f"scale must be positive and finite in fp32, got {given}")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    elif out.shape != shape or out.dtype != dtype or out.device != device or out.stride(2) != 1:
        raise ValueError("out must have q's shape, dtype and device, with a unit-stride head dim")
    o0, o1, _ = out.stride()
    if (B > 1 and o0 == 0) or (Hq > 1 and o1 == 0):
        raise ValueError("rows of out overlap")
    lse = q.new_empty((B, Hq), dtype=torch.float32) if return_lse else None
    w, w_strides, w_cols = _weights(cache, weights, B, pages)
    need = _decode_workspace(cache._geometry, B, Hq, pages, weights is not None)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.launch(
        device.index, "rp_paged_decode", cache._struct(), q.data_ptr(), _I64x2(q0, q1), _HALF[dtype], B, Hq,
        page_table.data_ptr(), row, pages, lengths.data_ptr(), 0.0 if scale is None else scale,
        out.data_ptr(), _I64x2(o0, o1), None if lse is None else lse.data_ptr(), w, w_strides, w_cols,
        ws.data_ptr(), need,
    )  # fmt: skip
    return (out, lse) if return_lse else out


class Evicted(NamedTuple):
    """``kept`` (sequences, heads, budget) int32 old positions in order, -1 past
    the end; ``lengths`` (sequences,) after the cut; ``weights`` (sequences,
    heads, positions of the new table) of the kept tokens, 0 past the end."""

    kept: torch.Tensor
    lengths: torch.Tensor
    weights: torch.Tensor


def evict(
    cache: PagedKV,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    weights: torch.Tensor,
    out_table: torch.Tensor,
    *,
    budget: int,
    recent: int,
) -> Evicted:
    """Cuts every sequence to at most ``budget`` tokens per KV head.

    A longer one keeps its last ``recent`` tokens and, of the older, the
    ``budget - recent`` of greatest accumulated weight (ties: the lowest
    position); a shorter one is kept whole.  The kept rows move, in order, to
    positions 0, 1, ... of ``out_table`` (sequences, pages), whose pages must
    be none of ``page_table``'s: nothing is written to those, which other
    sequences may share."""
    device = cache.device
    B, pages, row = _table(device, "page_table", page_table)
    _lengths(device, lengths, B)
    _, out_pages, out_row = _table(device, "out_table", out_table, B)
    budget, recent = int(budget), int(recent)
    if budget <= 0 or not 0 <= recent <= budget:
        raise ValueError(f"budget must be positive and recent in [0, budget], got {budget} and {recent}")
    if out_pages * cache.page_size < budget:
        raise ValueError(f"out_table holds {out_pages * cache.page_size} positions, the budget is {budget}")
    if weights is None:
        raise ValueError("evict needs the accumulated weights")
    w, w_strides, w_cols = _weights(cache, weights, B, pages)
    kept = lengths.new_empty((B, cache.heads, budget))
    new_lengths = torch.empty_like(lengths)
    new_weights = weights.new_empty((B, cache.heads, out_pages * cache.page_size))
    _lib.launch(
        device.index, "rp_paged_evict", cache._struct(), page_table.data_ptr(), row, pages, lengths.data_ptr(), B,
        w, w_strides, w_cols, out_table.data_ptr(), out_row, out_pages, budget, recent,
        kept.data_ptr(), new_lengths.data_ptr(), new_weights.data_ptr(),
    )  # fmt: skip
    return Evicted(kept, new_lengths, new_weights)


__all__ = ["Evicted", "HEAD_DIMS", "PagedKV", "alloc", "append", "decode", "evict"]
