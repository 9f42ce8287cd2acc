"""Rows of the softmax cross entropy far apart in memory, and single rows, whose stride is never walked."""
from __future__ import annotations

import ctypes as C

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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stride", [0, 5, 1 << 40])
@pytest.mark.parametrize("T,V", [(1, 300), (40, 1), (1, 1)])
def test_single_rows_of_a_description(ctx, T, V, stride, dtype):
    """The C description of one row or one item takes any stride for it, and so do their gradients."""
    from vectoraccelerate_amd import _lib

    D = 96
    h, w, y, _ = _inputs(T, V, D, dtype, T + V)
    loss, lse, mean = (torch.empty(n, device="cuda") for n in (T, T, 1))
    gh, gw = torch.empty_like(h), torch.empty_like(w)
    kinds = {torch.float32: _lib.VA_DTYPE_F32, torch.float16: _lib.VA_DTYPE_F16, torch.bfloat16: _lib.VA_DTYPE_BF16}
    hs, ws = stride if T == 1 else D, stride if V == 1 else D
    d = _lib.XentDesc(h.data_ptr(), w.data_ptr(), y.data_ptr(), None, hs, ws, IGNORE, T, V, D, kinds[dtype], 1.0)
    ctx.order_after_torch()
    ctx.check(ctx.lib.va_xent_forward(ctx.handle, C.byref(d), loss.data_ptr(), lse.data_ptr(), _lib.VA_REDUCE_MEAN, mean.data_ptr()), "va_xent_forward")
    ctx.check(ctx.lib.va_xent_backward(ctx.handle, C.byref(d), lse.data_ptr(), _lib.VA_REDUCE_MEAN, None, gh.data_ptr(), hs, gw.data_ptr(), ws),
              "va_xent_backward")
    ctx.synchronize()
    want = oracle.xent(h, w, y, 1.0, None, IGNORE, torch.full((T,), 1.0 / T, dtype=torch.float64))
    oracle.close(loss, *want["loss"], "loss")
    oracle.close(gh, *want["grad_hidden"], "grad_hidden")
    oracle.close(gw, *want["grad_items"], "grad_items")
