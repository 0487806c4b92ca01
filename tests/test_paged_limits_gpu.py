"""Calls of the paged operators at the limits of their arguments, on the GPU."""

from __future__ import annotations

import pytest
import torch
from test_paged_gpu import filled, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1e-46, 1e-300, 1e39, 0.0])
def test_a_scale_that_fp32_does_not_hold_is_refused(scale):
    """1e-46 rounds to 0 in fp32, which the library takes for 1 / sqrt(D)."""
    from repercep_runtime_b200 import paged

    cache, table, n, _, _ = filled([20, 3], 2, 16, 64, "bf16")
    q = rows((2, 4, 64), torch.bfloat16, 1)
    with pytest.raises(ValueError, match="scale"):
        paged.decode(q, cache, table, n, scale=scale)
    # the smallest normal value: all keys count alike
    weights = torch.zeros((2, 2, 32), device="cuda")
    paged.decode(q, cache, table, n, scale=2.0**-126, weights=weights)
    assert bool((weights[0, :, :20] == weights[0, 0, 0]).all())


def test_one_sequence_of_an_odd_pitch():
    """One token's q, k and v, whose tensors name an odd pitch between tokens."""
    from repercep_runtime_b200 import paged

    cache, table, n, _, _ = filled([20], 2, 16, 64, "bf16", width=2)
    wide = rows((8 * 64 + 5,), torch.bfloat16, 3)
    q, k, v = (wide.as_strided((1, h, 64), (517, 64, 1), at) for h, at in ((4, 0), (2, 256), (2, 384)))
    got = paged.append(cache, k, v, table, n)
    assert torch.equal(cache.k[int(table[0, 1]), :, 4], k[0])
    assert torch.equal(paged.decode(q, cache, table, got), paged.decode(q.clone(memory_format=torch.contiguous_format), cache, table, got))
