"""GPU parity of the paged attention where a call's arguments, not its sizes, are unusual.

References and tolerances are those of ``test_gpu_paged``.
"""

from __future__ import annotations

import math

import pytest
import torch

from granite_switch_amd import paged
from test_gpu_paged import BF16, FP32, Batch, _say

pytestmark = pytest.mark.gpu


# Chunks of more and of fewer than 16 rows, masked tails and diagonals; with 4100 cached tokens on
# few heads, tiles that are cut into parts.
SCALED = [("whole", [40, 1, 130, 3], [25, 70, 0, 300], 8, 2), ("cut", [40, 1, 130], [4100, 900, 3000], 4, 2)]


@pytest.mark.parametrize("scale", [4.0, 1e-3, 0.0, -1.0, -0.05])
@pytest.mark.parametrize("name,n,cached,heads,kv", SCALED, ids=[c[0] for c in SCALED])
@pytest.mark.parametrize("dim,window", [(128, 0), (64, 0), (80, 50)])
def test_ragged_scales(dev, scale, name, n, cached, heads, kv, dim, window):
    """A scale of zero weighs every key that a row sees alike; a negative one turns the order round."""
    _say(f"ragged scale {scale} {name} x {dim} window {window}")
    b = Batch(dev, n, cached, heads, kv, dim, seed=dim)
    lse = torch.empty(sum(n), heads, device=dev)
    out = b.run(scale=scale, window=window, lse=lse)
    torch.cuda.synchronize()
    b.check(out, scale=scale, window=window, lse=lse)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30])
def test_wide_windows(dev, dtype, window):
    """A window wider than any cache is none, for rows without a position too."""
    _say(f"window {window} {dtype}")
    b = Batch(dev, [40, 3, 20, 1], [-25, -3, 5, 200], 8, 2, 64, dtype=dtype, seed=9)
    out = b.run(window=window)
    torch.cuda.synchronize()
    b.check(out)
    assert torch.equal(out, b.run())
