"""Global gradient norm and clipping (va_clip.hip) against 64 bits: list lengths around a launch's, tensor sizes
around the vector and chunk edges, mixed types, alignment, in place and not, values without bound."""
from __future__ import annotations

import pytest
import torch

from tests import training_oracle as oracle
from tests.training_oracle import TINY, U, U32

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _tensors(sizes, types, seed, scale=0.01):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(types[i % len(types)]).cuda() for i, n in enumerate(sizes)]


def _check(ctx, tensors, max_norm, in_place=False, eps=1e-6):
    from vectoraccelerate_amd import GradientClipKernel

    k = GradientClipKernel(ctx)
    before = [t.cpu().double() for t in tensors]
    want = float(sum(float((b * b).sum()) for b in before)) ** 0.5
    norm = torch.full((1,), -1.0, device="cuda")
    outs = tensors if in_place else [torch.empty_like(t) for t in tensors]
    lst = k.tensorList(tensors, None if in_place else outs)
    ctx.order_after_torch()
    k.encode(lst, max_norm, norm, eps)
    ctx.synchronize()
    # fp64 sums: the norm is the rounding of the exact one; the factor one more, the product one
    oracle.close(norm, torch.tensor([want], dtype=torch.float64), torch.tensor([2 * U32 * want], dtype=torch.float64), "norm")
    f = min(1.0, max_norm / (want + eps))
    for o, b, t in zip(outs, before, tensors):
        oracle.close(o, b * f, (2 * U[t.dtype] + 4 * U32) * (b * f).abs() + TINY[t.dtype], f"tensor of {b.numel()}")
    return outs


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 255, 2048, 16_383, 16_384, 16_385, 40_000, 1_000_003])
@pytest.mark.parametrize("in_place", [False, True])
def test_one_tensor(ctx, n, dtype, in_place):
    _check(ctx, _tensors([n], [dtype], n), 0.05, in_place)


@pytest.mark.parametrize("count", [1, 2, 95, 96, 97, 193, 400])
def test_many_tensors_of_mixed_types(ctx, count):
    g = torch.Generator().manual_seed(count)
    sizes = torch.randint(1, 6000, (count,), generator=g).tolist()
    _check(ctx, _tensors(sizes, TYPES, count), 0.3)


def test_sizes_far_apart(ctx):
    """Some large tensors among empty and single-value ones."""
    sizes = [0, 1, 3_000_001, 0, 5, 17, 800_000] + [1] * 120 + [0, 2_000_000]
    _check(ctx, _tensors(sizes, TYPES, 3), 1.0)


def test_views_at_any_offset(ctx):
    flat = torch.randn(50_000, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    out = torch.zeros_like(flat)
    cuts = [0, 1, 4, 1003, 1004, 20_001, 49_999]
    from vectoraccelerate_amd import GradientClipKernel

    k = GradientClipKernel(ctx)
    a, b = ([t[i:j] for i, j in zip(cuts, cuts[1:])] for t in (flat, out))
    ctx.order_after_torch()
    k.encode(k.tensorList(a, b), 2.0)
    ctx.synchronize()
    x = flat.cpu().double()[: cuts[-1]]
    want = x * (2.0 / (float((x * x).sum()) ** 0.5 + 1e-6))
    oracle.close(out[: cuts[-1]], want, (2 * U[torch.bfloat16]) * want.abs(), "views")
    assert float(out[-1]) == 0.0


def test_nothing_to_clip(ctx):
    """A norm below the bound leaves every bit as it is."""
    t = _tensors([5000, 17, 40_001], TYPES, 5)
    for in_place in (False, True):
        before = [x.clone() for x in t]
        outs = _check(ctx, t, 1e6, in_place)
        assert all(torch.equal(o, b) for o, b in zip(outs, before))


def test_values_without_bound(ctx):
    """Squares beyond fp32's range, subnormals, infinities and NaN."""
    from vectoraccelerate_amd import GradientClipKernel

    k = GradientClipKernel(ctx)
    big = torch.full((1000,), 1e30, device="cuda")
    assert abs(k.clip([big], 1.0) / (1e30 * 1000**0.5) - 1) < 1e-6
    assert torch.allclose(big, torch.full_like(big, 1000**-0.5), rtol=1e-6)
    small = torch.full((1000,), 1e-30, device="cuda")
    assert abs(k.clip([small], 1.0) / (1e-30 * 1000**0.5) - 1) < 1e-5
    for v in (float("inf"), float("nan")):
        a, b = torch.ones(100, device="cuda"), torch.ones(70, device="cuda")
        a[7] = v
        n = k.clip([a, b], 1.0)
        if v == float("inf"):  # the factor is 0
            assert n == float("inf") and (b == 0).all() and torch.isnan(a[7])
        else:
            assert n != n and torch.isnan(a).all() and torch.isnan(b).all()


def test_empty_lists(ctx):
    from vectoraccelerate_amd import GradientClipKernel

    k = GradientClipKernel(ctx)
    assert k.clip([], 1.0) == 0.0
    assert k.clip([torch.empty(0, device="cuda"), torch.empty(0, device="cuda")], 1.0) == 0.0
    z = torch.zeros(10, device="cuda")
    assert k.clip([z], 1.0) == 0.0 and (z == 0).all()


def test_runs_agree_bit_for_bit(ctx):
    t = _tensors([100_000, 3, 70_001] * 40, TYPES, 9)
    a, b = _check(ctx, t, 0.2), _check(ctx, t, 0.2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals(ctx):
    from vectoraccelerate_amd import GradientClipKernel, VectorError

    k = GradientClipKernel(ctx)
    a = torch.ones(8, device="cuda")
    norm = torch.empty(1, device="cuda")
    for f in (lambda: k.tensorList([a.cpu()]), lambda: k.tensorList([a.double()]), lambda: k.tensorList([a.view(2, 4).T]), lambda: k.tensorList([a], []),
              lambda: k.tensorList([a], [a.half()]), lambda: k.tensorList([a], [a[:7]]), lambda: k.encode(k.tensorList([a]), -1.0, norm),
              lambda: k.encode(k.tensorList([a]), float("nan"), norm), lambda: k.encode(k.tensorList([a]), 1.0, norm.half()),
              lambda: k.encode(k.tensorList([a]), 1.0, norm, epsilon=-1.0)):
        with pytest.raises(VectorError):
            f()
