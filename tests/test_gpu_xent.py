"""Softmax cross entropy over a collection (va_xent.hip) against its definition in 64 bits: sizes around the
tile, stage and vector edges, every type, strides, offsets and masks, targets, reductions, streams."""
from __future__ import annotations

import pytest
import torch

from tests import training_oracle as oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
IGNORE = -100


def _inputs(T, V, D, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(T, D, generator=g)
    w = torch.randn(V, D, generator=g) * (spread / D**0.5)
    y = torch.randint(0, V, (T,), generator=g)
    return h.to(dtype).cuda(), w.to(dtype).cuda(), y.cuda(), g


def _check(ctx, h, w, y, scale=1.0, offsets=None, ignore=IGNORE, reduction="mean", up=None, backward=True):
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    k = SoftmaxCrossEntropyKernel(ctx)
    T, V = h.shape[0], w.shape[0]
    res = k.forward(h, w, y, reduction, scale, offsets, ignore)
    counted = (y != ignore).cpu()
    if reduction == "none":
        grad = up.cpu().double()
    else:
        grad = torch.full((T,), float(up) if up is not None else 1.0, dtype=torch.float64)
        if reduction == "mean":
            grad /= max(1, int(counted.sum()))
    want = oracle.xent(h, w, y, scale, offsets, ignore, grad)
    oracle.close(res.logSumExp, *want["lse"], "lse")
    oracle.close(res.loss, *want["loss"], "loss")
    if reduction != "none":
        loss, bound = want["loss"]
        n = max(1, int(counted.sum())) if reduction == "mean" else 1
        oracle.close(res.reduced, (loss[counted].sum() / n).view(1), (bound[counted].sum() / n + 2 * oracle.U32 * loss[counted].sum().abs() / n).view(1),
                     "reduced")
    if not backward:
        return res
    gh, gw = k.backward(h, w, y, res.logSumExp, up, reduction, scale, offsets, ignore)
    oracle.close(gh, *want["grad_hidden"], "grad_hidden")
    oracle.close(gw, *want["grad_items"], "grad_items")
    return res, gh, gw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 2, 3), (1, 1000, 64), (2, 257, 65), (7, 300, 7), (16, 512, 128), (17, 513, 96), (31, 700, 200),
                                   (33, 1025, 300), (63, 255, 63), (64, 256, 64), (65, 3000, 100), (100, 2000, 127), (128, 1024, 513),
                                   (255, 511, 72), (256, 768, 64), (257, 1300, 130), (300, 40, 768), (520, 2600, 40)])
def test_sizes(ctx, T, V, D, dtype):
    h, w, y, _ = _inputs(T, V, D, dtype, T * 7 + V + D)
    _check(ctx, h, w, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 5, 20, 50, 90, 150, 200])
def test_single_rows_to_many_over_a_long_collection(ctx, T, dtype):
    """More items than one round of every workgroup, a peaked softmax."""
    h, w, y, _ = _inputs(T, 70_001, 48, dtype, T, spread=3.0)
    _check(ctx, h, w, y, scale=2.5, backward=T < 60)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", [(260, 25_101, 520), (129, 49_200, 64), (513, 16_640, 300)])
def test_large_tiles(ctx, T, V, D, dtype):
    """Products of so many tiles that all of them take the largest."""
    h, w, y, g = _inputs(T, V, D, dtype, V)
    y[::7] = IGNORE
    off = torch.randn(V, generator=g)
    off[torch.rand(V, generator=g) < 0.1] = -torch.inf
    off[y.cpu().clamp(min=0)] = 0.5
    _check(ctx, h, w, y, scale=3.0, offsets=off.cuda())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D", [(3, 72), (70, 72), (220, 72), (3, 65), (70, 66), (220, 33)])
def test_offsets_and_masks(ctx, T, D, dtype):
    """Corrections; masked items that hold NaN and infinities; a masked target; the type's lowest value."""
    h, w, y, g = _inputs(T, 900, D, dtype, 11 + T)
    off = torch.randn(900, generator=g) * 2.0
    masked = torch.rand(900, generator=g) < 0.3
    masked[y.cpu()] = False
    off[masked] = -torch.inf
    w[masked.cuda()] = float("nan")
    w[int(torch.nonzero(masked)[0])] = float("inf")
    low = (~masked).nonzero().flatten()
    low = low[~torch.isin(low, y.cpu())][:5]
    off[low] = torch.finfo(torch.float32).min
    _check(ctx, h, w, y, scale=1.5, offsets=off.cuda())
    m = y.cpu()[0]
    off[m] = -torch.inf  # the target of row 0 (and of others perhaps) is deleted: loss +inf
    _check(ctx, h, w, y, offsets=off.cuda(), reduction="none", up=torch.ones(T, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [-torch.inf, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("T", [2, 80])
def test_every_item_masked(ctx, T, value, dtype):
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    h, w, y, _ = _inputs(T, 600, 64, dtype, 5)
    off = torch.full((600,), value, device="cuda")
    k = SoftmaxCrossEntropyKernel(ctx)
    res = k.forward(h, w, y, offsets=off)
    gh, gw = k.backward(h, w, y, res.logSumExp, offsets=off)
    if value == -torch.inf:
        assert torch.isneginf(res.logSumExp).all() and (res.loss == 0).all() and float(res.reduced) == 0.0
        assert (gh == 0).all() and (gw == 0).all()
    else:
        # every logit is the lowest value: lse is that too (log V is below its ulp), and everything is finite
        assert (res.logSumExp == value).all()
        assert torch.isfinite(res.loss).all() and torch.isfinite(gh).all() and torch.isfinite(gw).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D", [(6, 64), (130, 64), (40, 50), (260, 77)])
def test_ignored_and_invalid_targets(ctx, T, D, dtype):
    """Rows without a target hold NaN and infinities and change nothing; invalid targets give a NaN loss only."""
    h, w, y, _ = _inputs(T, 400, D, dtype, 3)
    y[::3] = IGNORE
    _check(ctx, h, w, y)
    y[1], y[2] = 400, -1
    _check(ctx, h, w, y, reduction="sum")
    y[1], y[2] = 3, 4
    clean = _check(ctx, h, w, y, reduction="sum")
    h[0], h[3] = float("nan"), float("inf")
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    k = SoftmaxCrossEntropyKernel(ctx)
    res = k.forward(h, w, y, "sum")
    gh, gw = k.backward(h, w, y, res.logSumExp, None, "sum")
    assert torch.equal(res.loss, clean[0].loss) and torch.equal(gh, clean[1]) and torch.equal(gw, clean[2])
    y[:] = IGNORE
    res = k.forward(h, w, y)
    gh, gw = k.backward(h, w, y, res.logSumExp)
    assert float(res.reduced) == 0.0 and (gh == 0).all() and (gw == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_upstream_gradients(ctx, reduction, dtype):
    """A scalar for a reduced loss; one a row, of either sign, zero and far apart, without a reduction."""
    h, w, y, g = _inputs(40, 300, 64, dtype, 17)
    if reduction == "none":
        up = torch.randn(40, generator=g) * torch.logspace(-3, 3, 40)
        up[5] = 0.0
        _check(ctx, h, w, y, reduction=reduction, up=up.cuda())
    else:
        _check(ctx, h, w, y, reduction=reduction, up=torch.tensor([-3.5], device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D,pad,shift", [(5, 64, 8, 0), (70, 64, 3, 0), (70, 128, 64, 1), (40, 50, 13, 1), (9, 50, 14, 2), (200, 70, 2, 0), (200, 33, 1, 0)])
def test_strided_and_misaligned_rows(ctx, T, D, pad, shift, dtype):
    """Rows within wider rows, starting off any alignment but the element's; what lies between is NaN."""
    h, w, y, _ = _inputs(T, 530, D, dtype, 23)

    def wide(m):
        flat = torch.full((m.shape[0] * (D + pad) + shift,), float("nan"), dtype=dtype, device="cuda")
        v = flat[shift:].view(m.shape[0], D + pad)[:, :D]
        v.copy_(m)
        return v

    a = _check(ctx, h, w, y)
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    k = SoftmaxCrossEntropyKernel(ctx)
    hw, ww = wide(h), wide(w)
    res = k.forward(hw, ww, y)
    gh, gw = wide(torch.zeros_like(h)), wide(torch.zeros_like(w))
    ctx.order_after_torch()
    k.encodeBackward(hw, ww, y, res.logSumExp, gh, gw)
    ctx.synchronize()
    _check(ctx, hw, ww, y)
    assert torch.equal(res.loss, a[0].loss) or torch.allclose(res.loss, a[0].loss, rtol=1e-5)
    base = gh._base if gh._base is not None else gh
    assert int(torch.isnan(base).sum()) == T * pad + shift, "values between the rows were written"
    grad = torch.full((T,), 1.0 / T, dtype=torch.float64)
    want = oracle.xent(h, w, y, 1.0, None, IGNORE, grad)
    oracle.close(gh, *want["grad_hidden"], "grad_hidden")
    oracle.close(gw, *want["grad_items"], "grad_items")


@pytest.mark.parametrize("dtype", TYPES)
def test_one_output_alone(ctx, dtype):
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    k = SoftmaxCrossEntropyKernel(ctx)
    h, w, y, _ = _inputs(90, 800, 96, dtype, 29)
    res, gh, gw = _check(ctx, h, w, y)
    a, b = torch.empty_like(gh), torch.empty_like(gw)
    ctx.order_after_torch()
    k.encodeBackward(h, w, y, res.logSumExp, a, None)
    k.encodeBackward(h, w, y, res.logSumExp, None, b)
    ctx.synchronize()
    assert torch.equal(a, gh) and torch.equal(b, gw)


@pytest.mark.parametrize("dtype", TYPES)
def test_runs_agree_bit_for_bit(ctx, dtype):
    """No result depends on the order in which workgroups run."""
    h, w, y, _ = _inputs(200, 5000, 64, dtype, 31)
    a, b = _check(ctx, h, w, y), _check(ctx, h, w, y)
    assert torch.equal(a[0].loss, b[0].loss) and torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("scale", [1.0, 4.0])
def test_gradients_against_differences(ctx, scale):
    """<gradient, v> against the central difference of the loss along v.  The step e leaves a term of e^2 / 6
    times the third derivative (below e^2 scale^3 for unit directions) and twice the loss's error over 2 e."""
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    k = SoftmaxCrossEntropyKernel(ctx)
    h, w, y, g = _inputs(30, 500, 64, torch.float32, 37)
    res, gh, gw = _check(ctx, h, w, y, scale=scale, reduction="sum")
    e = 2.0**-6
    for which in (0, 1):
        x = (h, w)[which]
        v = torch.randn(x.shape, generator=g).cuda()
        v /= v.norm()
        ends = [float(k.forward(*((x + s * e * v, w) if which == 0 else (h, x + s * e * v)), y, "sum", scale).loss.double().sum()) for s in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * e)
        got = float(((gh, gw)[which].double() * v.double()).sum())
        assert abs(slope - got) <= e * e * scale**3 * 30 + 2 * 30 * 2.0**-16 / (2 * e) * 0.1, (which, slope, got)


def test_rows_of_extreme_size_in_full_precision(ctx):
    """fp32 rows twelve decades apart: each row's logits keep the relative precision of its own values."""
    h, w, y, g = _inputs(24, 300, 64, torch.float32, 41)
    h *= torch.logspace(-6, 6, 24).cuda()[:, None]
    w *= torch.logspace(-9, 3, 300)[torch.randperm(300, generator=g)].cuda()[:, None]
    _check(ctx, h, w, y, scale=1e-6, backward=False)


def test_many_pieces(ctx):
    """A workspace that holds the items in several pieces gives what one piece gives (rows past 4,096 times
    the budget's items would; here the rows are many and the items few thousands)."""
    h, w, y, _ = _inputs(16_640, 33_000, 8, torch.bfloat16, 43)
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    k = SoftmaxCrossEntropyKernel(ctx)
    res = k.forward(h, w, y)
    gh, gw = k.backward(h, w, y, res.logSumExp)
    hd, wd = h.double(), w.double()
    z = hd @ wd.T
    lse = torch.logsumexp(z, 1)
    assert (res.logSumExp.double() - lse).abs().max() < 1e-4
    p = torch.exp(z - lse[:, None])
    p[torch.arange(p.shape[0], device="cuda"), y] -= 1.0
    p /= p.shape[0]
    for got, want in ((gh, p @ wd), (gw, p.T @ hd)):
        # both roundings to bf16 (2^-9 on average of a uniform mantissa) in the 2-norm
        assert (got.double() - want).norm() <= 2.0**-8 * want.norm()


def test_torch_stream_context(ctx):
    """A context on a stream of the caller's: calls queue behind its work and are complete in its order."""
    import ctypes as C

    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel, _lib

    h, w, y, _ = _inputs(50, 700, 64, torch.bfloat16, 47)
    want = _check(ctx, h, w, y)[0]
    stream = torch.cuda.Stream()
    handle = C.c_void_p()
    lib = _lib.load()
    assert lib.va_context_create_with_stream(0, C.c_void_p(stream.cuda_stream), C.byref(handle)) == 0

    class Borrowed:
        pass

    c = Borrowed()
    c.lib, c.handle, c.device = lib, handle, 0
    c.check = lambda st, what: (_ for _ in ()).throw(RuntimeError(what)) if st else None
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        h2 = (h.float() * 2).to(h.dtype) * 0.5
        loss, lse = torch.empty(50, device="cuda"), torch.empty(50, device="cuda")
        SoftmaxCrossEntropyKernel(c).encodeForward(h2, w, y, loss, lse)
        twice = loss * 2
    stream.synchronize()
    lib.va_context_destroy(handle)
    assert torch.equal(twice, want.loss * 2)


def test_refusals(ctx):
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel, VectorError

    k = SoftmaxCrossEntropyKernel(ctx)
    h, w, y, _ = _inputs(4, 10, 8, torch.float32, 1)
    loss, lse = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")

    def bad(kind="invalidInput", **kw):
        a = {"hidden": h, "items": w, "targets": y, "outLoss": loss, "outLogSumExp": lse} | kw
        with pytest.raises(VectorError) as e:
            k.encodeForward(**a)
        assert e.value.kind == kind, e.value

    bad(hidden=h.cpu())
    bad(hidden=h.double())
    bad(hidden=h.half())
    bad(hidden=h.flatten())
    bad("dimensionMismatch", items=w[:, :4].contiguous())
    bad(hidden=h.T.contiguous().T)
    bad(targets=y.int())
    bad(targets=y[:3])
    bad(outLoss=loss[:3])
    bad(outLoss=loss.half())
    bad(offsets=torch.zeros(9, device="cuda"))
    bad(scale=float("nan"))
    bad(outReduced=torch.empty(1, device="cuda"), reduction="none")
    bad(outReduced=torch.empty(1, device="cuda"), reduction="median")
    bad(hidden=h[:0], targets=y[:0], outLoss=loss[:0], outLogSumExp=lse[:0])
    bad(items=w[:0])
    gh, gw = torch.empty_like(h), torch.empty_like(w)
    for kw in ({"outGradHidden": None, "outGradItems": None}, {"outGradHidden": gh.half()}, {"outGradItems": gw[:5]}, {"reduction": "none"},
               {"reduction": "none", "grad": torch.ones(3, device="cuda")}, {"grad": torch.ones(4, device="cuda")},
               {"logSumExp": lse[:2]}):
        with pytest.raises(VectorError):
            k.encodeBackward(**({"hidden": h, "items": w, "targets": y, "logSumExp": lse, "outGradHidden": gh, "outGradItems": gw} | kw))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_rows_than_a_launch_holds(ctx, dtype):
    """Rows past what 2^23 workgroups of one launch take: a wave a row in the copies and at the loss's end."""
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    k = SoftmaxCrossEntropyKernel(ctx)
    T, V, D = (1 << 25) + 301, 3, 2
    g = torch.Generator("cuda").manual_seed(53)
    h = torch.randn(T, D, device="cuda", generator=g).to(dtype)
    w = torch.randn(V, D, device="cuda", generator=g).to(dtype)
    y = torch.randint(0, V, (T,), device="cuda", generator=g)
    res = k.forward(h, w, y, "none")
    for p in (slice(0, 400), slice((1 << 25) - 300, T)):
        want = oracle.xent(h[p], w, y[p], 1.0, None, IGNORE, torch.zeros(h[p].shape[0], dtype=torch.float64))
        oracle.close(res.logSumExp[p], *want["lse"], "lse")
        oracle.close(res.loss[p], *want["loss"], "loss")


def test_long_gradients_of_shares(ctx):
    """The hidden rows' gradient in shares of more values than a launch has threads."""
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    k = SoftmaxCrossEntropyKernel(ctx)
    T, V, D = (1 << 21) + 67, 700, 1028
    g = torch.Generator("cuda").manual_seed(59)
    h = torch.randn(T, D, device="cuda", dtype=torch.bfloat16, generator=g)
    w = torch.randn(V, D, device="cuda", dtype=torch.bfloat16, generator=g) * D**-0.5
    y = torch.randint(0, V, (T,), device="cuda", generator=g)
    res = k.forward(h, w, y, "sum")
    gh = torch.full_like(h, torch.nan)
    ctx.order_after_torch()
    k.encodeBackward(h, w, y, res.logSumExp, gh, None, None, "sum")
    ctx.synchronize()
    for p in (slice(0, 70), slice(T // 2, T // 2 + 70), slice(T - 70, T)):
        want = oracle.xent(h[p], w, y[p], 1.0, None, IGNORE, torch.ones(h[p].shape[0], dtype=torch.float64))
        oracle.close(gh[p], *want["grad_hidden"], "grad_hidden")
    assert not bool(torch.isnan(gh).any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", [(1, 1000, 768), (65, 129, 833), (64, 64, 1536), (30, 700, 2050), (130, 1900, 900), (5, 66, 5000)])
def test_few_tiles_with_many_stages(ctx, T, V, D, dtype):
    """Tiles whose stages are shared among waves, also when they do not divide evenly; with masks and both directions."""
    h, w, y, g = _inputs(T, V, D, dtype, T + V + D)
    off = torch.randn(V, generator=g)
    off[torch.rand(V, generator=g) < 0.1] = -torch.inf
    _check(ctx, h, w, y)
    _check(ctx, h, w, y, scale=0.5, offsets=off.cuda())


@pytest.mark.parametrize("T,V,D", [(1500, 12_000, 130), (1281, 30_001, 40)])
def test_large_tiles_of_planes(ctx, T, V, D):
    """fp32 rows and items that fill the chip with the largest tiles."""
    h, w, y, g = _inputs(T, V, D, torch.float32, T + V)
    off = torch.randn(V, generator=g)
    off[torch.rand(V, generator=g) < 0.05] = -torch.inf
    _check(ctx, h, w, y)
    _check(ctx, h, w, y, scale=0.7, offsets=off.cuda())


@pytest.mark.parametrize("dtype", TYPES)
def test_one_row_of_any_stride(ctx, dtype):
    """The stride of a single row is never walked: a view whose stride passes every limit is a row like any other."""
    h, w, y, _ = _inputs(1, 300, 96, dtype, 5)
    apart = h.as_strided((1, 96), (1 << 40, 1))
    _check(ctx, apart, w, y)
    _check(ctx, h.expand(1, 96).as_strided((1, 96), (0, 1)), w, y)
