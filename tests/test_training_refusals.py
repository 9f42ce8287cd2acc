"""Refusals of the training and serving operators that need no device: a NULL context at the C boundary, and
what the Python classes check before they call.  No kernel is launched here."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from vectoraccelerate_amd import GradientClipKernel, RMSNormKernel, SoftmaxCrossEntropyKernel, TensorList, VectorError, _lib


class NoDevice:
    """A context for calls that have to end before they reach it."""

    device = 0

    def __getattr__(self, name):
        raise AssertionError(f"the call went on to the context ({name})")


@pytest.fixture(scope="module")
def lib():
    from vectoraccelerate_amd import build as b

    if not _lib.LIB_PATH.exists():
        b.build()
    return _lib.load()


def test_null_context(lib):
    x, r, t = _lib.XentDesc(), _lib.RmsDesc(), _lib.TensorListDesc()
    assert lib.va_xent_forward(None, C.byref(x), None, None, 0, None) == 1
    assert lib.va_xent_backward(None, C.byref(x), None, 0, None, None, 0, None, 0) == 1
    assert lib.va_rms_norm(None, C.byref(r), None, 0) == 1
    assert lib.va_rms_norm_quantized(None, C.byref(r), 0, 0, 0.0, None, 0, None) == 1
    assert lib.va_rms_dequantize(None, None, 0, 0, None, 0.0, 1, 1, 0, 0, None, 0) == 1
    assert lib.va_rms_norm_backward(None, C.byref(r), None, 0, None, 0, None, None, 0, None) == 1
    assert lib.va_grad_clip(None, C.byref(t), 1.0, 0.0, None) == 1


def test_descriptions_match_the_header():
    """Sizes of the C structs on a 64-bit host."""
    assert C.sizeof(_lib.XentDesc) == 4 * 8 + 3 * 8 + 5 * 4 + 4
    assert C.sizeof(_lib.RmsDesc) == 5 * 8 + 3 * 8 + 4 * 4
    assert C.sizeof(_lib.TensorListDesc) == 4 * 8 + 8


def test_host_tensors_are_refused():
    c = NoDevice()
    x, w, y = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    out = torch.zeros(4)
    for f in (lambda: SoftmaxCrossEntropyKernel(c).encodeForward(x, w, y, out, out),
              lambda: SoftmaxCrossEntropyKernel(c).encodeForward(x.double(), w.double(), y, out, out),
              lambda: SoftmaxCrossEntropyKernel(c).encodeBackward(x, w, y, out, x, w),
              lambda: RMSNormKernel(c).encode(x, w[0], x),
              lambda: RMSNormKernel(c).encodeQuantized(x, w[0], x.to(torch.int8), out),
              lambda: RMSNormKernel(c).encodeDequantize(x.to(torch.int8), out, x),
              lambda: RMSNormKernel(c).encodeBackward(x, x, w[0], out, x),
              lambda: TensorList([x]), lambda: TensorList([x.double()]), lambda: TensorList([x], [])):
        with pytest.raises(VectorError):
            f()


def test_names_are_checked():
    with pytest.raises(VectorError):
        SoftmaxCrossEntropyKernel(NoDevice()).forward(torch.zeros(4, 8), None, None, reduction="total")
    assert GradientClipKernel(NoDevice()).tensorList([]).desc.count == 0
