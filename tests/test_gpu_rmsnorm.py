"""RMS norm with the residual's addition (va_rmsnorm.hip) against its definition in 64 bits: row lengths around
the vector, wave and workgroup edges, every type, 8-bit outputs, strides, in place, the backward pass."""
from __future__ import annotations

import pytest
import torch

from tests import training_oracle as oracle
from tests.training_oracle import TINY, U, U32

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
DIMS = [1, 7, 8, 9, 64, 127, 512, 513, 768, 1025, 1537, 2048, 2049, 4096, 4097, 8192, 8200, 20_001]
EPS = 1e-6


def _inputs(T, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + T * 31 + D)
    x, r = torch.randn(T, D, generator=g) * 2, torch.randn(T, D, generator=g)
    w = 1.0 + 0.3 * torch.randn(D, generator=g)
    return x.to(dtype).cuda(), r.to(dtype).cuda(), w.to(dtype).cuda(), g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("T,residual", [(1, True), (5, False), (9, True)])
def test_forward(ctx, T, D, residual, dtype):
    from vectoraccelerate_amd import RMSNormKernel

    x, r, w, _ = _inputs(T, D, dtype)
    y, s, inv = RMSNormKernel(ctx).forward(x, w, r if residual else None, EPS)
    rr, ii, yy, e = oracle.rms(x, r if residual else None, w, EPS)
    oracle.close(s, rr, U[dtype] * rr.abs() + TINY[dtype], "residual")
    oracle.close(inv, ii, e * ii, "inverse rms")
    oracle.close(y, yy, (e + U[dtype]) * yy.abs() + TINY[dtype], "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("group", [0, 8, 32, 128, 512])
@pytest.mark.parametrize("D", [1, 8, 100, 513, 768, 2048, 4100, 9001])
def test_codes(ctx, D, group, code, dtype):
    """Scales to rounding; a code is the nearest to y / s, or its neighbour where y / s lies within the
    arithmetic's error of the midpoint."""
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    T = 6
    x, r, w, _ = _inputs(T, D, dtype, 3)
    x[2], r[2] = 0.0, 0.0  # a row of zeros
    codes, scales, s = k.quantize(x, w, r, code, group, None, EPS)
    rr, ii, yy, e = oracle.rms(x, r, w, EPS)
    oracle.close(s, rr, U[dtype] * rr.abs() + TINY[dtype], "residual")
    most = 127.0 if code == torch.int8 else 448.0
    size = group or D
    groups = -(-D // size)
    z = torch.nn.functional.pad(yy, (0, groups * size - D)).view(T, groups, size)
    want = z.abs().amax(2) / most
    oracle.close(scales, want, (e + 2 * U32) * want, "scales")
    assert (scales[2] == 0).all()
    val = (z / want.clamp(min=1e-300).unsqueeze(2)).view(T, -1)[:, :D]
    got = codes.cpu().float().double()
    # half a step (int8: 1/2; e4m3: 2^-4 of the value, at least half of 2^-9), and the quotient's own error
    step = torch.full_like(val, 0.5) if code == torch.int8 else torch.maximum(val.abs() * 2.0**-4, torch.tensor(2.0**-10))
    assert ((got - val).abs() <= step + (2 * e + 8 * U32) * val.abs()).all()
    out = torch.empty(T, D, dtype=dtype, device="cuda")
    ctx.order_after_torch()
    k.encodeDequantize(codes, scales, out, group)
    ctx.synchronize()
    full = (codes.float().cpu() * scales.cpu().repeat_interleave(size, 1)[:, :D]).double()
    oracle.close(out, full, U[dtype] * full.abs() + TINY[dtype], "values")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("D", [96, 2500, 8300])
def test_given_scale_saturates(ctx, D, code, dtype):
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    x, r, w, _ = _inputs(4, D, dtype, 5)
    most = 127.0 if code == torch.int8 else 448.0
    given = 1.0 / most  # values past 1 saturate
    codes, scales, _ = k.quantize(x, w, r, code, 0, given, EPS)
    assert scales is None
    yy = oracle.rms(x, r, w, EPS)[2]
    got = codes.cpu().float().double()
    assert got.abs().max() == most
    sat = yy.abs() > 1.0 + 1e-4
    assert torch.equal(got[sat], most * yy[sat].sign())
    val = yy / given
    step = torch.full_like(val, 0.5) if code == torch.int8 else torch.maximum(val.abs() * 2.0**-4, torch.tensor(2.0**-10))
    inside = yy.abs() < 1.0
    assert ((got - val).abs() <= step + 1e-5 * val.abs())[inside].all()


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("group", [0, 32])
@pytest.mark.parametrize("D", [64, 8300])
def test_tiny_scales(ctx, D, group, code):
    """Scales below 2^-128, whose reciprocals are no fp32 values: zeros stay zeros, the others keep their codes."""
    from vectoraccelerate_amd import RMSNormKernel

    g = torch.Generator().manual_seed(D + group)
    x = torch.randn(3, D, generator=g) * 2e-37
    x[:, ::5] = 0.0
    w = torch.full((D,), 1e-4)
    codes, scales, _ = RMSNormKernel(ctx).quantize(x.cuda(), w.cuda(), None, code, group, None, EPS)
    _, _, yy, e = oracle.rms(x.cuda(), None, w.cuda(), EPS)
    most = 127.0 if code == torch.int8 else 448.0
    size = group or D
    groups = -(-D // size)
    z = torch.nn.functional.pad(yy, (0, groups * size - D)).view(3, groups, size)
    want = z.abs().amax(2) / most
    assert (want < 2.0**-128).all() and (want > 2.0**-140).all()
    # y and the scale are fp32 values below its normal ones: half of 2^-149 on top of the usual errors
    oracle.close(scales, want, (e + 2 * U32) * want + 2.0**-149, "scales")
    val = (z / want.unsqueeze(2)).view(3, -1)[:, :D]
    off = (2.0**-148 / want).repeat_interleave(size, 1)[:, :D]
    got = codes.cpu().float().double()
    assert torch.isfinite(got).all() and (got[:, ::5] == 0).all()
    step = torch.full_like(val, 0.5) if code == torch.int8 else torch.maximum(val.abs() * 2.0**-4, torch.tensor(2.0**-10))
    assert ((got - val).abs() <= step + (2 * e + 8 * U32 + off) * val.abs() + off).all()


@pytest.mark.parametrize("code", [None, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("D", [40, 3000, 9000])
def test_non_finite_rows_stay_alone(ctx, D, code):
    """NaN or inf in one row makes that row's values NaN and no other's."""
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    x, _, w, _ = _inputs(5, D, torch.float32, 7)
    clean = k.forward(x, w)[0] if code is None else k.quantize(x, w, None, code)[:2]
    x[1, D // 2], x[3, 0] = float("nan"), float("inf")
    keep = [0, 2, 4]
    if code is None:
        y = k.forward(x, w)[0]
        assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[1]).all() and torch.isnan(y[3, 0])
        return
    codes, scales = k.quantize(x, w, None, code)[:2]
    assert torch.equal(codes.view(torch.int8)[keep], clean[0].view(torch.int8)[keep]) and torch.equal(scales[keep], clean[1][keep])
    assert not torch.isfinite(scales[[1, 3]]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [60, 513, 2304, 9000])
def test_strided_and_in_place(ctx, D, dtype):
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    x, r, w, _ = _inputs(7, D, dtype, 9)
    y, s, inv = k.forward(x, w, r)
    wide = [torch.full((7, D + 5), float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
    xs, rs = (t[:, 3 : 3 + D] for t in wide)
    xs.copy_(x)
    rs.copy_(r)
    ctx.order_after_torch()
    k.encode(xs, w, xs, rs, rs, None)
    ctx.synchronize()
    assert torch.equal(xs, y) and torch.equal(rs, s)
    assert all(int(torch.isnan(t).sum()) == 35 for t in wide)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("T,extra", [(1, False), (6, True), (1030, True)])
def test_backward(ctx, T, D, extra, dtype):
    if T * D > 10_000_000:
        T = 40
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    x, r, w, g = _inputs(T, D, dtype, 13)
    dy = torch.randn(T, D, generator=g).to(dtype).cuda()
    dr = torch.randn(T, D, generator=g).to(dtype).cuda() if extra else None
    _, s, inv = k.forward(x, w, r, EPS)
    gx, gw = k.backward(dy, s, w, inv, dr)
    S, W, G = s.cpu().double(), w.cpu().double(), dy.cpu().double()
    i = inv.cpu().double()[:, None]
    n = S * i
    along = (G * W * n).mean(1, keepdim=True)
    want = i * (G * W - n * along) + (dr.cpu().double() if extra else 0.0)
    # `along` is a sum of D products (48 u32 of their magnitudes); four operations follow
    mag = i * ((G * W).abs() + n.abs() * (G * W * n).abs().mean(1, keepdim=True)) + (dr.cpu().double().abs() if extra else 0.0)
    oracle.close(gx, want, 64 * U32 * mag + 2 * U[dtype] * want.abs() + TINY[dtype], "grad_x")
    gwant = (G * n).sum(0)
    # T products in chains of at most T / 512 + 64 and a tree
    oracle.close(gw, gwant, (T / 512 + 80) * U32 * (G * n).abs().sum(0) + U[dtype] * gwant.abs() + TINY[dtype], "grad_weight")


def test_backward_against_differences(ctx):
    """<gradient, v> against the central difference of sum(dy y) along v, evaluated in 64 bits from the
    kernel's definition (the forward kernel is tested against that)."""
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    x, _, w, g = _inputs(8, 300, torch.float32, 17)
    dy = torch.randn(8, 300, generator=g).cuda()
    _, s, inv = k.forward(x, w, None, EPS)
    gx, gw = k.backward(dy, s, w, inv)
    e = 1e-4

    def value(xx, ww):
        return float((dy.cpu().double() * oracle.rms(xx, None, ww, EPS)[2]).sum())

    v, u = torch.randn(8, 300, generator=g).double(), torch.randn(300, generator=g).double()
    xd, wd = x.cpu().double(), w.cpu().double()
    dx = (value(xd + e * v, wd) - value(xd - e * v, wd)) / (2 * e)
    dw = (value(xd, wd + e * u) - value(xd, wd - e * u)) / (2 * e)
    assert abs(dx - float((gx.cpu().double() * v).sum())) < 1e-4
    assert abs(dw - float((gw.cpu().double() * u).sum())) < 1e-3


@pytest.mark.parametrize("D", [700, 9000])
def test_one_gradient_alone(ctx, D):
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    x, _, w, g = _inputs(33, D, torch.bfloat16, 19)
    dy = torch.randn(33, D, generator=g).bfloat16().cuda()
    _, s, inv = k.forward(x, w)
    gx, gw = k.backward(dy, s, w, inv)
    a, b = torch.empty_like(gx), torch.empty_like(gw)
    ctx.order_after_torch()
    k.encodeBackward(dy, s, w, inv, a, None)
    k.encodeBackward(dy, s, w, inv, None, b)
    ctx.synchronize()
    assert torch.equal(a, gx) and torch.equal(b, gw)


def test_refusals(ctx):
    from vectoraccelerate_amd import RMSNormKernel, VectorError

    k = RMSNormKernel(ctx)
    x, r, w, _ = _inputs(4, 32, torch.float32)
    codes, scales = torch.empty(4, 32, dtype=torch.int8, device="cuda"), torch.empty(4, 1, device="cuda")
    for f in (lambda: k.encode(x.cpu(), w, x), lambda: k.encode(x.double(), w.double(), x.double()), lambda: k.encode(x, w[:31], x),
              lambda: k.encode(x, w.half(), x), lambda: k.encode(x, w, x[:3]), lambda: k.encode(x, w, x.half()),
              lambda: k.encode(x, w, x, residual=r[:, :16]), lambda: k.encode(x, w, x, epsilon=-1.0), lambda: k.encode(x, w, x, epsilon=float("nan")),
              lambda: k.encode(x[:0], w, x[:0]), lambda: k.encode(x.T.contiguous().T, w, x),
              lambda: k.encodeQuantized(x, w, codes.float(), scales), lambda: k.encodeQuantized(x, w, codes, None),
              lambda: k.encodeQuantized(x, w, codes, scales, givenScale=0.1), lambda: k.encodeQuantized(x, w, codes, None, givenScale=-0.1),
              lambda: k.encodeQuantized(x, w, codes, torch.empty(4, 2, device="cuda"), groupSize=24),
              lambda: k.encodeQuantized(x, w, codes, scales, groupSize=16), lambda: k.encodeDequantize(codes, scales, x[:2]),
              lambda: k.encodeBackward(x, x, w, torch.empty(3, device="cuda"), x), lambda: k.encodeBackward(x, x, w, torch.empty(4, device="cuda"))):
        with pytest.raises(VectorError):
            f()


@pytest.mark.parametrize("code", [None, torch.int8])
def test_more_rows_than_a_launch_holds(ctx, code):
    """Rows past what one launch's 2^23 workgroups take (and a launch's 2^32 threads would)."""
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    T, D = (1 << 26) + 77, 3
    x = torch.randn(T, D, device="cuda", dtype=torch.bfloat16, generator=torch.Generator("cuda").manual_seed(5))
    w = torch.tensor([1.0, -0.5, 2.0], device="cuda", dtype=torch.bfloat16)
    parts = [slice(0, 500), *(slice((i << 25) - 500, (i << 25) + 500) for i in (1, 2)), slice(T - 300, T)]
    if code is None:
        y, _, inv = k.forward(x, w, None, EPS)
        for p in parts:
            _, ii, yy, e = oracle.rms(x[p], None, w, EPS)
            oracle.close(inv[p], ii, e * ii, "inverse rms")
            oracle.close(y[p], yy, (e + U[torch.bfloat16]) * yy.abs() + TINY[torch.bfloat16], "y")
        return
    codes, scales, _ = k.quantize(x, w)
    y = torch.empty(T, D, device="cuda", dtype=torch.float32)
    k.encodeDequantize(codes, scales, y)
    ctx.synchronize()
    for p in parts:
        _, ii, yy, e = oracle.rms(x[p], None, w, EPS)
        want = yy.abs().amax(1) / 127.0
        oracle.close(scales[p].squeeze(1), want, (e + 2 * U32) * want, "scales")
        # (half a step of the code and what the arithmetic moves y / s by; the product's own rounding)
        oracle.close(y[p], yy, want[:, None] * (0.5 + 127.0 * (2 * e + 8 * U32)), "codes")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [700, 3000, 9000])
@pytest.mark.parametrize("over", ["grad", "residual", "x"])
def test_backward_in_place(ctx, D, dtype, over):
    """The gradient of x written over one of the operands."""
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    T = 40
    x, r, w, g = _inputs(T, D, dtype, 29)
    dy, dr = (torch.randn(T, D, generator=g).to(dtype).cuda() for _ in range(2))
    _, s, inv = k.forward(x, w, r)
    gx, gw = k.backward(dy, s, w, inv, dr)
    out, weight = {"grad": dy, "residual": dr, "x": s}[over], torch.empty_like(gw)
    ctx.order_after_torch()
    k.encodeBackward(dy, s, w, inv, out, weight, dr)
    ctx.synchronize()
    assert torch.equal(out, gx) and torch.equal(weight, gw)
