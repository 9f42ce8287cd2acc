"""Calls of the training kernels give the same bits again, whatever the outputs and the scratch memory held."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,V,D,dtype,masks", [(1023, 49_999, 300, torch.float16, False), (1500, 60_000, 384, torch.bfloat16, True), (300, 30_000, 200, torch.float32, True),
                                               (12, 50_000, 768, torch.bfloat16, False), (50, 90_000, 130, torch.float32, False), (10, 5000, 513, torch.float32, True)])
def test_cross_entropy(ctx, T, V, D, dtype, masks):
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    k = SoftmaxCrossEntropyKernel(ctx)
    g = torch.Generator("cuda").manual_seed(T)
    h, w = (torch.randn(n, D, device="cuda", generator=g).to(dtype) * D**-0.25 for n in (T, V))
    y = torch.randint(0, V, (T,), device="cuda", generator=g)
    y[::9] = -100
    off = None
    if masks:
        off = torch.randn(V, device="cuda", generator=g)
        off[::50] = -torch.inf
        w[::50] = torch.inf
    runs = []
    for fill in (torch.nan, 1.0, -3.0):
        out = [torch.full(s, fill, device="cuda", dtype=t) for s, t in (((T,), torch.float32), ((T,), torch.float32), ((1,), torch.float32), ((T, D), dtype), ((V, D), dtype))]
        torch.cuda.synchronize()
        k.encodeForward(h, w, y, *out[:3], offsets=off)
        k.encodeBackward(h, w, y, out[1], out[3], out[4], offsets=off)
        # something else in the scratch memory before the next run
        k.forward(h[: T // 2 + 1].float() * fill, w[:777].float(), y[: T // 2 + 1].clamp(max=776))
        ctx.synchronize()
        runs.append(out)
    assert not any(bool(torch.isnan(o).any()) for o in runs[0])
    for out in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], out))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,D", [(10_007, 513), (3000, 3000), (700, 9000)])
def test_rms_norm(ctx, T, D, dtype):
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    g = torch.Generator("cuda").manual_seed(T)
    x, r, dy, dr = (torch.randn(T, D, device="cuda", generator=g).to(dtype) for _ in range(4))
    w = torch.randn(D, device="cuda", generator=g).to(dtype)
    runs = []
    for fill in (torch.nan, 1.0):
        y, s, gx = (torch.full_like(x, fill) for _ in range(3))
        gw, inv, scales = torch.full_like(w, fill), torch.full((T,), fill, device="cuda"), torch.full((T, -(-D // 64)), fill, device="cuda")
        codes = torch.full((T, D), 99, device="cuda", dtype=torch.int8)
        torch.cuda.synchronize()
        k.encode(x, w, y, r, s, inv)
        k.encodeQuantized(x, w, codes, scales, r, None, None, 64)
        k.encodeBackward(dy, s, w, inv, gx, gw, dr)
        ctx.synchronize()
        runs.append((y, s, gx, gw, inv, scales, codes))
    assert not any(bool(torch.isnan(o.float()).any()) for o in runs[0])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_clipping(ctx):
    from vectoraccelerate_amd import GradientClipKernel

    k = GradientClipKernel(ctx)
    g = torch.Generator("cuda").manual_seed(1)
    tensors = [torch.randn(n, device="cuda", generator=g).bfloat16() for n in [1_000_003, 17, 30_000_001] + [9000] * 200]
    runs = []
    for fill in (torch.nan, 1.0):
        outs, norm = [torch.full_like(t, fill) for t in tensors], torch.full((1,), fill, device="cuda")
        torch.cuda.synchronize()
        k.encode(k.tensorList(tensors, outs), 1.0, norm)
        ctx.synchronize()
        runs.append([norm, *outs])
    assert not any(bool(torch.isnan(o).any()) for o in runs[0])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_ordered_by_streams_alone(ctx):
    """The context's stream waits for torch's and torch's for it, on the device: a step without a host synchronisation."""
    from vectoraccelerate_amd import GradientClipKernel, RMSNormKernel, SoftmaxCrossEntropyKernel

    norm, entropy, clip = RMSNormKernel(ctx), SoftmaxCrossEntropyKernel(ctx), GradientClipKernel(ctx)
    g = torch.Generator("cuda").manual_seed(2)
    T, V, D = 500, 4000, 128
    x, items, w = torch.randn(T, D, device="cuda", generator=g), torch.randn(V, D, device="cuda", generator=g) * 0.1, torch.ones(D, device="cuda")
    y = torch.randint(0, V, (T,), device="cuda", generator=g)

    def step(order):
        a, b = order
        h, dh, gx, gi, inv = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(items), torch.empty(T, device="cuda")
        loss, lse, mean, total = (torch.empty(n, device="cuda") for n in (T, T, 1, 1))
        slow = torch.randn(3000, 3000, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
        for _ in range(8):
            slow = slow @ slow * 1e-2  # torch's stream is behind when the calls are queued
        xx = x * 2.0 + slow[0, 0] * 0.0
        a()
        norm.encode(xx, w, h, outInverseRms=inv)
        entropy.encodeForward(h, items, y, loss, lse, mean)
        entropy.encodeBackward(h, items, y, lse, dh, gi)
        norm.encodeBackward(dh, xx, w, inv, gx)
        clip.encode(clip.tensorList([gi, gx]), 0.01, total)
        b()
        out = [t * 1.0 for t in (mean, total, gi, gx)]
        torch.cuda.synchronize()
        ctx.synchronize()
        return out

    here, there = torch.cuda.current_stream(), ctx.torch_stream()
    want = step((ctx.order_after_torch, ctx.synchronize))
    got = step((lambda: there.wait_stream(here), lambda: here.wait_stream(there)))
    assert all(torch.equal(p, q) for p, q in zip(want, got))
