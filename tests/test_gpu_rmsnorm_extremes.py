"""RMS norm of rows whose squares pass fp32's range or fall below it, though the rows and results are ordinary values."""
from __future__ import annotations

import pytest
import torch

from tests import training_oracle as oracle
from tests.training_oracle import TINY, U, U32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [3, 64, 768, 2000, 2304, 8192, 9001])
@pytest.mark.parametrize("size,eps", [(-110, 0.0), (-70, 0.0), (-52, 1e-30), (62, 1e-6), (66, 1e-6), (120, 1e-6)])
def test_sizes(ctx, D, size, eps, dtype):
    """Rows of 2^size: forward, codes and backward; among them one of zeros and one of ordinary size."""
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    g = torch.Generator().manual_seed(D + size)
    x = torch.randn(7, D, generator=g) * 2.0**size
    x[2] = torch.randn(D, generator=g)
    x = x.to(dtype).cuda()
    w = (1.0 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda()
    y, _, inv = k.forward(x, w, None, eps)
    _, ii, yy, e = oracle.rms(x, None, w, eps)
    oracle.close(inv, ii, e * ii, "inverse rms")
    oracle.close(y, yy, (e + U[dtype]) * yy.abs() + TINY[dtype], "y")
    codes, scales, _ = k.quantize(x, w, None, torch.int8, 0, None, eps)
    want = yy.abs().amax(1, keepdim=True) / 127.0
    oracle.close(scales, want, (e + 2 * U32) * want, "scales")
    assert bool(((codes.cpu().double() - yy / want).abs() <= 0.5 + 127.0 * (2 * e + 8 * U32)).all())
    dy = torch.randn(7, D, generator=g).to(dtype).cuda()
    gx, _ = k.backward(dy, x, w, inv)
    i = inv.cpu().double()[:, None]
    n, gy = x.cpu().double() * i, dy.cpu().double() * w.cpu().double()
    want = i * (gy - n * (gy * n).mean(1, keepdim=True))
    mag = i * (gy.abs() + n.abs() * (gy * n).abs().mean(1, keepdim=True))
    oracle.close(gx, want, 64 * U32 * mag + 2 * U[dtype] * want.abs() + 2.0**-126, "grad_x")


@pytest.mark.parametrize("D", [64, 768, 2304, 9001])
def test_rows_of_zeros(ctx, D):
    """With an epsilon, zeros are normed to zeros beside rows of any size."""
    from vectoraccelerate_amd import RMSNormKernel

    x = torch.zeros(5, D)
    x[1], x[3] = 1e30, 1e-30
    w = torch.ones(D)
    y, _, inv = RMSNormKernel(ctx).forward(x.cuda(), w.cuda(), None, 1e-6)
    _, ii, yy, e = oracle.rms(x, None, w, 1e-6)
    oracle.close(inv, ii, e * ii, "inverse rms")
    oracle.close(y, yy, (e + U32) * yy.abs() + TINY[torch.float32], "y")
