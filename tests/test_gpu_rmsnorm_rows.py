"""RMS norm backward of so many rows that every wave or workgroup takes several, the next one's loads in flight."""
from __future__ import annotations

import pytest
import torch

from tests.training_oracle import TINY, U, U32

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _near(got, want, bound, name):
    off = ~((got.double() - want).abs() <= bound)
    assert not bool(off.any()), f"{name}: {int(off.sum())} of {off.numel()} off"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D", [(10_007, 7), (10_007, 513), (10_007, 768), (9001, 2048), (5003, 2304), (5003, 4096), (3001, 8192), (1201, 9001)])
@pytest.mark.parametrize("over", [None, "grad", "residual", "x"])
def test_many_rows(ctx, T, D, dtype, over):
    """Both gradients, apart from the operands and written over each of them."""
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    g = torch.Generator("cuda").manual_seed(T + D)
    r, dy, dr = (torch.randn(T, D, device="cuda", generator=g).to(dtype) for _ in range(3))
    w = (1.0 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(dtype)
    R, G, W, extra = r.double(), dy.double(), w.double(), dr.double() if over != "x" else 0.0
    inv = (1.0 / torch.sqrt((R * R).mean(1) + 1e-6)).float()
    out = {None: torch.full_like(r, torch.nan), "grad": dy, "residual": dr, "x": r}[over]
    gw = torch.full_like(w, torch.nan)
    ctx.order_after_torch()
    k.encodeBackward(dy, r, w, inv, out, gw, dr if over != "x" else None)
    ctx.synchronize()
    i = inv.double()[:, None]
    n = R * i
    want = i * (G * W - n * (G * W * n).mean(1, keepdim=True)) + extra
    # the mean of D products is off by 48 u32 of their magnitudes, four operations follow
    mag = i * ((G * W).abs() + n.abs() * (G * W * n).abs().mean(1, keepdim=True)) + (extra.abs() if over != "x" else 0.0)
    _near(out, want, 64 * U32 * mag + 2 * U[dtype] * want.abs() + TINY[dtype], "grad_x")
    gwant = (G * n).sum(0)
    _near(gw, gwant, (T / 256 + 80) * U32 * (G * n).abs().sum(0) + U[dtype] * gwant.abs() + TINY[dtype], "grad_weight")
