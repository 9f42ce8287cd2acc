"""Rows of the softmax cross entropy far apart in memory."""
from __future__ import annotations

import pytest
import torch

from tests import training_oracle as oracle
from tests.test_gpu_xent import IGNORE, TYPES, _check, _inputs

pytestmark = pytest.mark.gpu


def _apart(m, stride):
    """The rows of m `stride` elements apart in a buffer of their own; what lies between is not set."""
    flat = torch.empty((m.shape[0] - 1) * stride + m.shape[1], dtype=m.dtype, device="cuda")
    v = flat.as_strided(m.shape, (stride, 1))
    v.copy_(m)
    return v


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D", [(5, 64), (40, 70), (70, 64), (200, 72)])
@pytest.mark.parametrize("which", ["hidden", "items", "both"])
def test_rows_megabytes_apart(ctx, T, D, which, dtype):
    """Strides of 12 MB, as the last position of each of many sequences has them: in, and for the gradients out."""
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    h, w, y, g = _inputs(T, 90, D, dtype, T + D)
    off = torch.zeros(90)
    off[::9] = -torch.inf
    off[y.cpu()] = 0.0
    stride = (12 << 20) // h.element_size() + (2 if D == 64 else 1)
    hh = _apart(h, stride) if which != "items" else h
    ww = _apart(w, stride) if which != "hidden" else w
    _check(ctx, hh, ww, y)
    res = _check(ctx, hh, ww, y, offsets=off.cuda())[0]
    k = SoftmaxCrossEntropyKernel(ctx)
    gh, gw = (_apart(torch.zeros_like(m), stride) for m in (h, w))
    ctx.order_after_torch()
    k.encodeBackward(hh, ww, y, res.logSumExp, gh, gw, offsets=off.cuda())
    ctx.synchronize()
    want = oracle.xent(h, w, y, 1.0, off.cuda(), IGNORE, torch.full((T,), 1.0 / T, dtype=torch.float64))
    oracle.close(gh, *want["grad_hidden"], "grad_hidden")
    oracle.close(gw, *want["grad_items"], "grad_items")
