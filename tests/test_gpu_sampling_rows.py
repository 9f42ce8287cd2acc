"""Rows that the passes over them give up on, in the first pass and in the second, beside rows that they take, divided among
workgroups (va_sample.hip); against the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_sampling import _check, _kernel, _logits

pytestmark = pytest.mark.gpu


def _given_up(V):
    """Rows of which the second pass finds more items at the cut than a list holds (equal ones, of one and of two values, and a
    plateau below a peak), the first no item in its sample, and ordinary ones."""
    x, u = _logits(8, V, torch.float32, V)
    x[0] = 0.5
    x[1] = -2.0
    x[1, ::2] = -2.25
    x[2] = -3.0
    x[2, V // 2 : V // 2 + 20] = 1.0
    x[3] = -torch.inf
    x[3, V // 3] = 4.0
    x[4] = torch.nan
    return x, u


@pytest.mark.parametrize("V", [70_000, 1 << 18])
@pytest.mark.parametrize("s", [dict(topK=20_000), dict(topP=0.4), dict(topP=0.7, topK=30_000), dict(topP=0.9, minP=0.001), dict(topK=10_000, minP=0.0001)])
def test_rows_that_the_second_pass_gives_up_on(ctx, V, s):
    x, u = _given_up(V)
    _check(ctx, x, u, **s)
    k, x, u = _kernel(ctx), x.cuda(), u.cuda()
    want = k.sample(x, u, **s)
    for _ in range(10):
        got = k.sample(x, u, **s)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1].view(torch.int32), want[1].view(torch.int32))
