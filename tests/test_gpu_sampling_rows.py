"""Rows that the passes over them give up on, in the first pass and in the second, beside rows that they take, divided among
workgroups (va_sample.hip); against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
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


def _first_kept(x, temperature, topK, topP, minP):
    """The first kept item that weighs anything in fp64, of one row: what u = 0 draws in the order of the items; and its share."""
    x = np.asarray(x, np.float64)
    items = np.nonzero(x > -np.inf)[0]
    items = items[np.lexsort((items, -x[items]))]
    w = np.exp((x[items] - x[items[0]]) / temperature)
    upto = np.cumsum(w)
    n = min(topK or len(items), len(items))
    if topP < 1:
        n = min(n, int(np.searchsorted(upto, topP * upto[n - 1])) + 1)
    n = min(n, int((w >= minP).sum()))
    first = int(items[:n][w[:n] > 0].min())
    return first, float(np.exp((x[first] - x[items[0]]) / temperature) / upto[n - 1])


@pytest.mark.parametrize("V", [1500, 9000, 40_000, 300_000])
@pytest.mark.parametrize("s", [dict(), dict(temperature=0.5), dict(topK=1000), dict(topK=3000), dict(topK=200, topP=0.9999), dict(topP=0.9), dict(topP=1 - 2.0**-24), dict(minP=1e-30), dict(topK=100, minP=1e-20)])
def test_nothing_random_draws_the_first_kept_item(ctx, V, s):
    """u = 0 draws the first kept item, little as it may weigh: 2^-701 of the largest, items that do so together where none does alone,
    below 2^-51 of a list's largest, and behind masked ones."""
    g = torch.Generator().manual_seed(V)
    x = torch.full((7, V), -torch.inf)
    x[0, 1:512] = -486.0
    x[0, 700] = 0.0
    x[1, 5] = -486.1
    x[1, 1400:] = torch.randn(V - 1400, generator=g)
    x[2, 9:] = torch.randn(V - 9, generator=g) - 40.0
    x[2, 1300:1340] = torch.randn(40, generator=g)
    x[3] = torch.randn(V, generator=g)
    x[3, :3] = -torch.inf
    x[4, 7:600] = -480.0 - torch.rand(593, generator=g) * 30
    x[4, V - 1] = 3.0
    x[5, 3:] = -36.0
    x[5, 600:900] = torch.rand(300, generator=g)
    x[6, 100:] = -300.0
    x[6, V - 300 :] = 1.0
    settings = dict(temperature=1.0, topK=0, topP=1.0, minP=0.0) | s
    items, logs = (t.cpu().tolist() for t in _kernel(ctx).sample(x.cuda(), torch.zeros(7, device="cuda"), **s))
    settings["topP"], settings["minP"] = float(np.float32(settings["topP"])), float(np.float32(settings["minP"]))
    for t in range(7):
        want, share = _first_kept(x[t].double().numpy(), **settings)
        assert items[t] == want, f"row {t}: item {items[t]} where {want} is right"
        assert abs(logs[t] - np.log(share)) <= 2.0**-22 * abs(np.log(share)) + 1e-10, f"row {t}"


@pytest.mark.parametrize("V", [900, 10_000, 50_000])
def test_fewer_items_than_top_k_keeps(ctx, V):
    """Masked rows: one item left, some, as many as top-k keeps, one more; in either order of the draw."""
    from tests.test_gpu_sampling_order import _check as check_falling

    x, u = _logits(24, V, torch.float32, V)
    g = torch.Generator().manual_seed(V)
    for t, left in enumerate([1, 2, 3, 40, 49, 50, 51, 64, 65, 300, 500, 850] * 2):
        x[t, torch.randperm(V, generator=g)[left:]] = -torch.inf if t < 12 else torch.nan
    for s in (dict(topK=50), dict(topK=300, topP=0.9), dict(topK=600, minP=0.01), dict(topK=899), dict(topK=50, topP=0.5, minP=0.1)):
        _check(ctx, x, u, **s)
        check_falling(ctx, x, u, **s)


@pytest.mark.parametrize("V", [2000, 300_000])
def test_a_share_below_the_least_number(ctx, V):
    """An item far below the row's largest, which no sample meets: if u = 0 draws it, its log probability is finite and its own."""
    x = torch.zeros(3, V)
    x[:, 0] = torch.tensor([-430.0, -600.0, -690.0])
    x[:, 1711] = torch.tensor([600.0, 400.0, 620.0])
    items, logs = (t.cpu().tolist() for t in _kernel(ctx).sample(x.cuda(), torch.zeros(3, device="cuda")))
    for t in range(3):
        a = x[t].double()
        want = float(a[items[t]] - torch.logsumexp(a, 0))
        assert items[t] in (0, 1) and abs(logs[t] - want) <= 2.0**-22 * abs(want), f"row {t}: {items[t]}, {logs[t]} where {want} is right"
