"""Masked items of the softmax cross entropy that hold large finite values: a sum of their products overflows
although none of them is NaN or inf, and still they have no probability and no gradient."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_xent import TYPES, _check, _inputs

pytestmark = pytest.mark.gpu

# few rows, a middling product, and one of so many tiles that all of them take the largest
SHAPES = [(3, 300, 72), (70, 900, 65), (200, 700, 128), (513, 16_640, 64)]


def _masked(V, y, g):
    masked = torch.rand(V, generator=g) < 0.1
    masked[y.cpu()] = False
    return masked, torch.zeros(V).masked_fill(masked, -torch.inf).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", SHAPES)
def test_largest_finite_values(ctx, T, V, D, dtype):
    """+, - and either sign of the type's largest value, against ordinary hidden rows."""
    h, w, y, g = _inputs(T, V, D, dtype, T + D)
    masked, off = _masked(V, y, g)
    most = torch.finfo(dtype).max
    sign = torch.where(torch.rand(V, D, generator=g) < 0.5, -1.0, 1.0)
    sign[::3] = 1.0
    sign[1::3] = -1.0
    w[masked.cuda()] = (sign * most).to(dtype).cuda()[masked.cuda()]
    _check(ctx, h, w, y, scale=1.5, offsets=off)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,V,D", SHAPES)
@pytest.mark.parametrize("size", [50, 70, 100])
def test_large_hidden_rows(ctx, T, V, D, size, dtype):
    """Hidden rows of 2^size, items as much smaller but for the masked ones, which are middling."""
    h, w, y, g = _inputs(T, V, D, dtype, T + D + size)
    masked, off = _masked(V, y, g)
    h, w = h * 2.0**size, w * 2.0**-size
    w[masked.cuda()] = 2.0 ** (130 - size)
    _check(ctx, h, w, y, offsets=off)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V", [(1, 60), (10, 900), (40, 300), (70, 130)])
@pytest.mark.parametrize("stages", [5, 9, 10, 12, 13, 14, 15, 17, 18, 22, 25, 34])
def test_rows_next_to_masked_ones(ctx, T, V, stages, dtype):
    """Rows whose last 128 bytes are begun by a single dword and continued by the next item's, which is masked and holds NaN
    or inf; tiles of so many stages that groups of waves share them, in any remainder."""
    D = (stages - 1) * 32 + 1
    if dtype != torch.float32:
        D *= 2
    h, w, y, g = _inputs(T, V, D, dtype, T + D)
    masked, off = _masked(V, y, g)
    w[masked.cuda()] = torch.inf
    w[torch.nonzero(masked)[::2].flatten().cuda()] = torch.nan
    _check(ctx, h, w, y, offsets=off)
