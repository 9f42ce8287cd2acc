"""Gradients of the softmax cross entropy over the whole range of a type: small probabilities, rows of very unlike size
and upstream gradients far apart, with bounds that are relative to each result's own terms."""
from __future__ import annotations

import pytest
import torch

from tests.training_oracle import U, U32, close

pytestmark = pytest.mark.gpu

# on both sides of where fp32 rows stop being multiplied as they are
ROWS = [20, 32, 33, 64, 65, 100, 300]


def _gradients(h, w, y, scale, g):
    """Both gradients in 64 bits and their bounds, for the row gradients g [T] (float64) and targets within the items.

    A logit is off by the roundings of its products and their sum: D u32 of the magnitudes, 2^-20 of them where fp32
    values are two fp16 values each, and then (a value far below its row's largest is off by 2^-39 of that) D 2^-38
    of the two rows' largest; 4 u32 of itself for the factor and the difference with lse.  lse is off by as much, 2^-16
    for the sum of the exponentials and 4 u32 of itself.  dl = g (p - [target]) is off by p times both, by its own
    rounding, and by the smallest exponential, 2^-126.  Sums of n terms in fp32 are off by n u32 of the magnitudes."""
    dtype = h.dtype
    T, V, D = h.shape[0], w.shape[0], h.shape[1]
    h, w, y = h.cpu().double(), w.cpu().double(), y.cpu()
    z = scale * (h @ w.T)
    lse = torch.logsumexp(z, 1)
    full = dtype == torch.float32
    ez = abs(scale) * ((D + 4) * U32 + (2.0**-20 if full else 0.0)) * (h.abs() @ w.abs().T) + 4 * U32 * z.abs()
    if full:
        ez += abs(scale) * D * 2.0**-38 * h.abs().amax(1)[:, None] * w.abs().amax(1)[None, :]
    e_lse = ez.amax(1) + 2.0**-16 + 4 * U32 * lse.abs()
    p = torch.exp(z - lse[:, None])
    d = p.clone()
    d[torch.arange(T), y] -= 1.0
    dl = g[:, None] * d
    rounding = (4 * U32) if full else U[dtype] + 4 * U32
    edl = g.abs()[:, None] * (p * (ez + e_lse[:, None]) + 2.0**-126) + dl.abs() * rounding
    s = abs(scale)
    gh, gw = scale * (dl @ w), scale * (dl.T @ h)
    e_gh = s * (edl @ w.abs()) + (V + 8) * U32 * s * (dl.abs() @ w.abs()) + 2 * U[dtype] * gh.abs() + 2.0**-126
    e_gw = s * (edl.T @ h.abs()) + (T + 8) * U32 * s * (dl.abs().T @ h.abs()) + 2 * U[dtype] * gw.abs() + 2.0**-126
    return (gh, e_gh), (gw, e_gw)


def _check(ctx, h, w, y, scale, reduction="mean", up=None):
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    k = SoftmaxCrossEntropyKernel(ctx)
    res = k.forward(h, w, y, reduction, scale)
    gh, gw = k.backward(h, w, y, res.logSumExp, up, reduction, scale)
    T = h.shape[0]
    g = up.cpu().double() if reduction == "none" else torch.full((T,), 1.0 / T, dtype=torch.float64)
    (want_h, e_h), (want_w, e_w) = _gradients(h, w, y, scale, g)
    close(gh, want_h, e_h, "grad_hidden")
    close(gw, want_w, e_w, "grad_items")


def _unit_rows(T, V, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    h, w = torch.randn(T, D, generator=g), torch.randn(V, D, generator=g)
    h, w = h / h.norm(dim=1, keepdim=True), w / w.norm(dim=1, keepdim=True)
    y = torch.randint(0, V, (T,), generator=g)
    return h.to(dtype).cuda(), w.to(dtype).cuda(), y.cuda(), g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 20.0, 30.0, 50.0, 100.0])
@pytest.mark.parametrize("T", ROWS)
def test_small_probabilities(ctx, T, scale, dtype):
    """Unit rows at inverse temperatures up to 100: most items have probabilities far below 2^-38, and a gradient."""
    h, w, y, _ = _unit_rows(T, 4000, 96, dtype, T)
    _check(ctx, h, w, y, scale)


@pytest.mark.parametrize("T", ROWS)
@pytest.mark.parametrize("D", [64, 130])
@pytest.mark.parametrize("which", ["hidden", "both"])
def test_rows_of_extreme_size(ctx, T, D, which):
    """fp32 rows twelve decades apart, the smallest with logits of about 1; and items twelve decades apart beside them."""
    h, w, y, g = _unit_rows(T, 1500, D, torch.float32, T + D)
    h *= torch.logspace(-6, 6, T)[torch.randperm(T, generator=g)].cuda()[:, None]
    w *= 1e6 if which == "hidden" else torch.logspace(-9, 3, 1500)[torch.randperm(1500, generator=g)].cuda()[:, None]
    _check(ctx, h, w, y, 3.0 if which == "hidden" else 1e-6)


@pytest.mark.parametrize("T", ROWS)
def test_upstream_gradients_far_apart(ctx, T):
    """fp32 rows whose upstream gradients are sixteen decades apart, each row's own gradient in full."""
    h, w, y, g = _unit_rows(T, 2000, 64, torch.float32, T)
    up = torch.logspace(-10, 6, T)[torch.randperm(T, generator=g)] * torch.where(torch.rand(T, generator=g) < 0.5, -1.0, 1.0)
    _check(ctx, h, w, y, 10.0, "none", up.cuda())


@pytest.mark.parametrize("T,V,D", [(1500, 12_000, 130), (400, 30_001, 72), (40, 70_000, 64)])
def test_small_probabilities_of_larger_products(ctx, T, V, D):
    """The same where tiles are of other sizes and sums are shared among workgroups."""
    h, w, y, _ = _unit_rows(T, V, D, torch.float32, T + V)
    _check(ctx, h, w, y, 40.0)
