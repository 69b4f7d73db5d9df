"""Residual norm where a call's sizes are unusual."""

from __future__ import annotations

import pytest
import torch

from granite_switch_amd import norms

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(4, 0), (0, 64), (0, 0), (2, 3, 0)])
def test_nothing_to_do(dev, shape):
    """A call without elements gives empty results, and does so again (its checks are kept by layout)."""
    print(f"norm {shape}", flush=True)
    x, r, w = torch.zeros(shape, device=dev), torch.zeros(shape, device=dev), torch.ones(shape[-1], device=dev)
    for _ in range(3):
        y, ro = norms.residual_norm(x, r, w)
        assert y.shape == ro.shape == shape
