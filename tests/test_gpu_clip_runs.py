"""Gradient clipping where a workgroup takes runs of chunks, across tensors' ends, and around a launch's list."""
from __future__ import annotations

import pytest
import torch

from tests.training_oracle import TINY, U, U32

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _check(ctx, sizes, max_norm, in_place, seed):
    """As the tensors of test_gpu_clip, with the definition in 64 bits on the device."""
    from vectoraccelerate_amd import GradientClipKernel

    g = torch.Generator("cuda").manual_seed(seed)
    # every tensor of its own size: a chunk taken from another tensor, twice or not at all shows in the norm
    tensors = [(torch.randn(n, device="cuda", generator=g) * (0.01 + 0.003 * (i % 11))).to(TYPES[i % 3]) for i, n in enumerate(sizes)]
    before = [t.double() for t in tensors]
    want = float(torch.stack([(b * b).sum() for b in before]).sum()) ** 0.5
    outs = tensors if in_place else [torch.full_like(t, torch.nan) for t in tensors]
    norm = torch.full((1,), -1.0, device="cuda")
    k = GradientClipKernel(ctx)
    ctx.order_after_torch()
    k.encode(k.tensorList(tensors, None if in_place else outs), max_norm, norm)
    ctx.synchronize()
    # fp64 sums: the norm is the rounding of the exact one; the factor one more, the product one
    assert abs(float(norm) - want) <= 2 * U32 * want
    f = min(1.0, max_norm / (want + 1e-6))
    for i, (o, b) in enumerate(zip(outs, before)):
        e = (2 * U[o.dtype] + 4 * U32) * (b * f).abs() + TINY[o.dtype]
        assert bool(((o.double() - b * f).abs() <= e).all()), (i, o.numel())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("count,most", [(60, 2_000_000), (1, 45_000_001), (170, 500_000), (700, 100_000)])
def test_runs_of_chunks(ctx, count, most, in_place):
    """More chunks than the chip holds workgroups (about 1800 of 16,384 values), in tensors of uneven sizes."""
    sizes = [most] if count == 1 else torch.randint(1, most, (count,), generator=torch.Generator().manual_seed(count)).tolist()
    assert sum(sizes) > 30_000_000
    _check(ctx, sizes, 0.5, in_place, count)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("count", [165, 166, 167, 331, 332, 333])
def test_lists_around_a_launch(ctx, count, in_place):
    sizes = torch.randint(1, 40_000, (count,), generator=torch.Generator().manual_seed(count)).tolist()
    _check(ctx, sizes, 0.5, in_place, count)


def test_empty_tensors_between_launches(ctx):
    """Empty tensors count for no launch's list, wherever they stand."""
    _check(ctx, [0] * 200 + [5] * 166 + [0] * 3 + [20_000] * 166 + [0] * 40 + [7], 0.5, False, 1)
