"""Scores of sampled tokens on B200 (librepercep_b200.so).

The reference's token-VLA planner decodes candidate action chunks and ranks
them (``VLAEngine.plan``, src/repercep/models/vla.py:229-258).
``token_logprobs`` gives what such a ranking needs from the logits in one pass:
the log probability of each sampled token, the entropy of its distribution,
and the top alternatives.

Torch allocates the outputs and supplies the current stream; the arithmetic
runs in the library, which has no fallback (a missing library raises).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

MAX_TOP = 64
_LOGITS = {
    torch.bfloat16: _lib.RP_DTYPE_BF16,
    torch.float16: _lib.RP_DTYPE_F16,
    torch.float32: _lib.RP_DTYPE_F32,
}


class TokenScores(NamedTuple):
    """Per row: ``logprobs`` and ``entropy`` fp32 (rows,), ``top_logprobs`` fp32
    and ``top_ids`` int64 (rows, top), largest first, ties to the lowest id."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_ids: torch.Tensor


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenScores:
    """Scores ``tokens`` (rows,) int64 under ``logits`` (rows, vocab) bf16, fp16
    or fp32 (any row stride, unit-stride vocabulary).

    A negative token marks a row without one: its log probability is 0.
    ``top`` (0..64, at most vocab) alternatives come with every row."""
    if logits.dim() != 2:
        raise ValueError("logits must be 2-D (rows, vocab)")
    if logits.dtype not in _LOGITS:
        raise ValueError(f"logits must be bf16, fp16 or fp32, got {logits.dtype}")
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor")
    rows, vocab = logits.shape
    if vocab == 0:
        raise ValueError("logits have an empty vocabulary")
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("logits must have a unit-stride vocabulary")
    device = logits.device
    if tokens.dtype != torch.int64 or tokens.shape != (rows,) or tokens.device != device:
        raise ValueError(f"tokens must be int64 ({rows},) on {device}")
    if rows > 1 and tokens.stride(0) != 1:
        raise ValueError("tokens must be contiguous")
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be in [0, {min(MAX_TOP, vocab)}], got {top}")
    logprobs = logits.new_empty(rows, dtype=torch.float32)
    entropy = torch.empty_like(logprobs)
    top_logprobs = logprobs.new_empty((rows, top))
    top_ids = tokens.new_empty((rows, top))
    args = (
        logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, _LOGITS[logits.dtype], rows, vocab,
        tokens.data_ptr(), top, logprobs.data_ptr(), entropy.data_ptr(), top_logprobs.data_ptr(), top_ids.data_ptr(),
    )  # fmt: skip
    _lib.launch(device.index, "rp_token_logprobs", *args)
    return TokenScores(logprobs, entropy, top_logprobs, top_ids)


__all__ = ["MAX_TOP", "TokenScores", "token_logprobs"]
