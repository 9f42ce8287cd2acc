"""Rows and dimensions past what the RMS norm's kernels count in 32 bits are refused before anything is launched."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim", [(1, 0xFFFFFFFF), (2, 0xFFFFFFF9), (1, 0x7FFFFFFF), (0xFFFFFFFF, 8), (0x80000000, 1)])
def test_sizes_past_the_limits(ctx, rows, dim):
    from vectoraccelerate_amd import VectorError, _lib

    x = torch.zeros(64, device="cuda")
    p, far, lib, h = x.data_ptr(), 1 << 33, ctx.lib, ctx.handle
    d = _lib.RmsDesc(p, None, p, None, None, far, 0, 0, rows, dim, _lib.VA_DTYPE_F32, 1e-6)
    for name, call in (("va_rms_dequantize", lambda: lib.va_rms_dequantize(h, p, far, _lib.VA_CODE_INT8, p, 0.0, rows, dim, 0, _lib.VA_DTYPE_F32, p, far)),
                       ("va_rms_norm", lambda: lib.va_rms_norm(h, C.byref(d), p, far)),
                       ("va_rms_norm_quantized", lambda: lib.va_rms_norm_quantized(h, C.byref(d), _lib.VA_CODE_INT8, 0, 0.0, p, far, p)),
                       ("va_rms_norm_backward", lambda: lib.va_rms_norm_backward(h, C.byref(d), p, far, None, 0, p, p, far, p))):
        with pytest.raises(VectorError) as e:
            ctx.check(call(), name)
        assert e.value.kind == "invalidInput" and "too many" in str(e.value)
