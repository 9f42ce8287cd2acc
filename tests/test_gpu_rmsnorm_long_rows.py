"""RMS norm of rows of up to millions of values: sums as exact as those of short rows, and the limits of a row."""
from __future__ import annotations

import pytest
import torch

from tests import training_oracle as oracle
from tests.training_oracle import TINY, U, U32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [8193, 100_003, 1 << 20, (1 << 22) + 5])
def test_sums(ctx, D, dtype):
    """The inverse rms is off by half of the mean's roundings (its sum in 64 bits, one quotient, one addition) and by
    its own (root and quotient): 4 u32, and the product with the row and the weight by 2 more.  The gradient's mean of products
    carries 3 u32 of each, two operations and the result follow."""
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    g = torch.Generator().manual_seed(D)
    # values of one sign and of nearly one size: a chain of fp32 additions rounds them alike
    x = (1.1 + 0.01 * torch.randn(3, D, generator=g)).to(dtype).cuda()
    w = (1.0 + 0.1 * torch.randn(D, generator=g)).to(dtype).cuda()
    dy = (0.7 + 0.01 * torch.randn(3, D, generator=g)).to(dtype).cuda()
    y, _, inv = k.forward(x, w, None, 1e-6)
    _, ii, yy, _ = oracle.rms(x, None, w, 1e-6)
    oracle.close(inv, ii, 4 * U32 * ii, "inverse rms")
    oracle.close(y, yy, (6 * U32 + U[dtype]) * yy.abs() + TINY[dtype], "y")
    gx, gw = k.backward(dy, x, w, inv)
    i = inv.cpu().double()[:, None]
    n, gy = x.cpu().double() * i, dy.cpu().double() * w.cpu().double()
    want = i * (gy - n * (gy * n).mean(1, keepdim=True))
    mag = i * (gy.abs() + n.abs() * (gy * n).abs().mean(1, keepdim=True))
    oracle.close(gx, want, 8 * U32 * mag + 2 * U[dtype] * want.abs() + TINY[dtype], "grad_x")
    gwant = (dy.cpu().double() * n).sum(0)
    oracle.close(gw, gwant, 8 * U32 * (dy.cpu().double() * n).abs().sum(0) + U[dtype] * gwant.abs(), "grad_weight")


def test_codes_of_long_rows(ctx):
    """The codes of a long row from the same sums."""
    from vectoraccelerate_amd import RMSNormKernel

    D = (1 << 20) + 3
    x = (1.1 + 0.01 * torch.randn(2, D, generator=torch.Generator().manual_seed(1))).cuda()
    w = torch.ones(D, device="cuda")
    _, scales, _ = RMSNormKernel(ctx).quantize(x, w, None, torch.int8)
    want = oracle.rms(x, None, w, 1e-6)[2].abs().amax(1, keepdim=True) / 127.0
    oracle.close(scales, want, 8 * U32 * want, "scales")


def test_weight_gradient_of_more_values_than_a_launch_has_threads(ctx):
    """A row of so many values that the sum of its weight's gradient takes more threads than a launch can have."""
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    D = (1 << 28) + 1021
    g = torch.Generator("cuda").manual_seed(3)
    x, dy = (torch.randn(1, D, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    w = torch.ones(D, device="cuda", dtype=torch.bfloat16)
    inv = torch.full((1,), 0.75, device="cuda")
    gw = torch.full_like(w, torch.nan)
    ctx.order_after_torch()
    k.encodeBackward(dy, x, w, inv, None, gw)
    ctx.synchronize()
    want = (dy.float() * (x.float() * 0.75))[0]
    assert not bool(torch.isnan(gw).any())
    # one product in fp32 before the rounding, in the kernel and here
    assert bool(((gw.float() - want).abs() <= 2 * U[torch.bfloat16] * want.abs() + TINY[torch.bfloat16]).all())
