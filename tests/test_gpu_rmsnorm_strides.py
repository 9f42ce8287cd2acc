"""Single rows of the RMS norm: their stride in the C description is never walked."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from tests import training_oracle as oracle
from tests.training_oracle import TINY, U, U32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stride", [0, 3, 1 << 40])
@pytest.mark.parametrize("D", [96, 3000, 9000])
def test_single_rows_of_a_description(ctx, D, stride):
    from vectoraccelerate_amd import _lib

    g = torch.Generator().manual_seed(D)
    x, r, dy, dr = (torch.randn(1, D, generator=g).bfloat16().cuda() for _ in range(4))
    w = torch.randn(D, generator=g).bfloat16().cuda()
    s, y, gx, back = (torch.empty_like(x) for _ in range(4))
    gw, inv, scale = torch.empty_like(w), torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    codes = torch.empty(1, D, dtype=torch.int8, device="cuda")
    d = _lib.RmsDesc(x.data_ptr(), r.data_ptr(), w.data_ptr(), s.data_ptr(), inv.data_ptr(), stride, stride, stride, 1, D, _lib.VA_DTYPE_BF16, 1e-6)
    b = _lib.RmsDesc(s.data_ptr(), None, w.data_ptr(), None, None, stride, 0, 0, 1, D, _lib.VA_DTYPE_BF16, 0.0)
    lib, h = ctx.lib, ctx.handle
    ctx.order_after_torch()
    ctx.check(lib.va_rms_norm(h, C.byref(d), y.data_ptr(), stride), "va_rms_norm")
    ctx.check(lib.va_rms_norm_quantized(h, C.byref(d), _lib.VA_CODE_INT8, 0, 0.0, codes.data_ptr(), stride, scale.data_ptr()), "va_rms_norm_quantized")
    ctx.check(lib.va_rms_dequantize(h, codes.data_ptr(), stride, _lib.VA_CODE_INT8, scale.data_ptr(), 0.0, 1, D, 0, _lib.VA_DTYPE_BF16, back.data_ptr(), stride),
              "va_rms_dequantize")
    ctx.check(lib.va_rms_norm_backward(h, C.byref(b), dy.data_ptr(), stride, dr.data_ptr(), stride, inv.data_ptr(), gx.data_ptr(), stride, gw.data_ptr()),
              "va_rms_norm_backward")
    ctx.synchronize()
    rr, ii, yy, e = oracle.rms(x, r, w, 1e-6)
    oracle.close(s, rr, U[x.dtype] * rr.abs() + TINY[x.dtype], "residual")
    oracle.close(y, yy, (e + U[x.dtype]) * yy.abs() + TINY[x.dtype], "y")
    step = yy.abs().amax(1, keepdim=True) / 127.0
    oracle.close(back, yy, step * (0.5 + 127.0 * (2 * e + 8 * U32)) + U[x.dtype] * yy.abs(), "codes")
    n = s.cpu().double() * inv.cpu().double()[:, None]
    G, W = dy.cpu().double(), w.cpu().double()
    want = inv.cpu().double()[:, None] * (G * W - n * (G * W * n).mean(1, keepdim=True)) + dr.cpu().double()
    mag = inv.cpu().double()[:, None] * ((G * W).abs() + n.abs() * (G * W * n).abs().mean(1, keepdim=True)) + dr.cpu().double().abs()
    oracle.close(gx, want, 64 * U32 * mag + 2 * U[x.dtype] * want.abs(), "grad_x")
    oracle.close(gw, (G * n)[0], (4 * U32 + U[x.dtype]) * (G * n)[0].abs(), "grad_weight")
