"""Rows near the ends of fp32's range whose logits are ordinary numbers."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_xent import _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,V,D", [(20, 700, 64), (70, 900, 65), (200, 700, 128), (1500, 12_000, 40)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [-115, -108, -60, 60, 115])
def test_sizes_that_cancel(ctx, T, V, D, size, dtype):
    """Hidden rows of 2^size and items of 2^-size."""
    h, w, y, g = _inputs(T, V, D, dtype, T + D)
    h, w = h * 2.0**size, w * 2.0**-size
    off = torch.randn(V, generator=g)
    off[::7] = -torch.inf
    off[y.cpu()] = 0.0
    _check(ctx, h, w, y)
    _check(ctx, h, w, y, offsets=off.cuda())
