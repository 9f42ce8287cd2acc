"""Drawing along falling logits (va_sample.hip, order "logits") against the definition in 64 bits: every kind of cut, lists from the top and
from the middle, draws that need a list of their own, ties, masks, rows that the passes give up on, graphs and workspaces."""
from __future__ import annotations

import ctypes as C
import subprocess

import numpy as np
import pytest
import torch

from tests.test_gpu_sampling import LAST, SETTINGS, TYPES, _kernel, _logits, _rows
from tests.test_gpu_sampling_rows import _given_up

pytestmark = pytest.mark.gpu


def drawn(x, u, temperature, k, p, m):
    """(item, probability, how far the draw is from the next border as a share of the sum) of one row, in 64 bits."""
    x = np.asarray(x, np.float64) + 0.0
    items = np.nonzero(~np.isnan(x) & (x > -np.inf))[0]
    if not len(items):
        return -1, 0.0, 1.0
    items = items[np.lexsort((items, -x[items]))]
    v = x[items]
    if temperature == 0:
        k, temperature = 1, 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(v == v[0], 1.0, np.exp((v - v[0]) / temperature))
    upto = np.cumsum(w)
    n = min(k, len(items)) if k else len(items)
    near = 1.0
    if p < 1:
        total = upto[n - 1]
        by = int(np.searchsorted(upto, p * total)) + 1
        near = min(near, *(abs(upto[j] / total - p) for j in range(max(0, by - 2), min(by + 1, len(upto)))))
        n = min(n, by)
    if m > 0:
        near = min(near, float(np.abs(w / m - 1)[w != 1.0].min(initial=1.0)))
        n = min(n, int((w >= m).sum()))
    total = upto[n - 1]
    at = min(int(np.searchsorted(upto[:n], u * total, side="right")), n - 1, int(np.nonzero(w)[0][-1]))
    near = min(near, float(np.abs(upto[:n] / total - u).min()))
    if np.isin(w, (0.0, 1.0)).all():  # sums of whole numbers are exact
        near = 1.0
    return int(items[at]), w[at] / total, near


def _check(ctx, logits, u, temperature=1.0, topK=0, topP=1.0, minP=0.0):
    """A draw nearer than 2^-40 to a border may fall on either side (fp64's sums of up to a million weights: 2^20 times 2^-53 at most,
    and the weights' own 2^-44)."""
    k = _kernel(ctx)
    dev = lambda v: v.cuda() if isinstance(v, torch.Tensor) else v  # noqa: E731
    items, logs = k.sample(logits.cuda(), u.cuda(), dev(temperature), dev(topK), dev(topP), dev(minP), order="logits")
    items, logs = items.cpu().tolist(), logs.cpu().double().tolist()
    T = logits.shape[0]
    x = logits.double().numpy()
    settings = [_rows(v.double() if isinstance(v, torch.Tensor) and v.dtype == torch.float32 else v, T) for v in (temperature, topK, topP, minP)]
    f = lambda v: float(np.float32(v))  # noqa: E731
    unclear = 0
    for t in range(T):
        want, probability, near = drawn(x[t], float(u[t]), f(settings[0][t]), int(settings[1][t]), f(settings[2][t]), f(settings[3][t]))
        if near < 2.0**-40:
            unclear += 1
            continue
        assert items[t] == want, f"row {t}: item {items[t]} where {want} is right"
        if want < 0:
            assert logs[t] == -np.inf
        else:
            assert abs(logs[t] - np.log(probability)) <= 2.0**-23 * abs(np.log(probability)) + 1e-10, f"row {t}"
    assert unclear <= max(1, T // 100)
    return items


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("s", range(len(SETTINGS)))
def test_settings(ctx, s, dtype):
    for T, V in ((40, 1000), (40, 20_000), (20, 60_000)):
        _check(ctx, *_logits(T, V, dtype, s), **SETTINGS[s])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 3, 64, 65, 511, 512, 513, 1025, 4095, 4097, 8193, 24_575, 24_577, 65_537, 131_073])
def test_sizes(ctx, V, dtype):
    for i, s in enumerate((dict(), dict(topK=20, topP=0.9), dict(topP=0.95, temperature=0.8), dict(minP=0.05), dict(minP=1e-5))):
        _check(ctx, *_logits(3, V, dtype, V + i), **s)


@pytest.mark.parametrize("T", [1, 2, 63, 255, 257, 1023, 1025])
def test_numbers_of_rows(ctx, T):
    for V in (3000, 25_000) if T < 300 else (3000,):
        _check(ctx, *_logits(T, V, torch.float32, T), topP=0.9)
        _check(ctx, *_logits(T, V, torch.bfloat16, T), topK=30)
        _check(ctx, *_logits(T, V, torch.float16, T))


def test_more_long_rows_than_share_a_launch(ctx):
    x, u = _logits(16, 30_000, torch.float16, 1)
    T = 1030
    x, u = x.repeat(65, 1)[:T].contiguous(), torch.rand(T, generator=torch.Generator().manual_seed(2))
    _check(ctx, x, u, topP=0.8, temperature=2.0)


# flat rows, whose nuclei are thousands of items: the draw falls above the list that holds the cut
WIDE = [dict(topP=0.5), dict(topP=0.9), dict(topP=0.99, temperature=1.5), dict(topP=0.9, minP=0.3), dict(topP=0.9, minP=0.02), dict(minP=0.1), dict(minP=0.5, temperature=2.0),
        dict(topP=0.9, minP=0.9), dict(topK=3000), dict(topK=4097, topP=0.7), dict()]


@pytest.mark.parametrize("s", range(len(WIDE)))
@pytest.mark.parametrize("T,V", [(5, 16_000), (6, 100_003), (2, 700_001)])
def test_wide_nuclei(ctx, T, V, s):
    for dtype, spread in ((torch.float32, 0.3), (torch.float16, 0.5), (torch.bfloat16, 1.0)):
        g = torch.Generator().manual_seed(s)
        x = (torch.randn(T, V, generator=g) * spread).to(dtype)
        for u in (torch.rand(T, generator=g), torch.linspace(0.0, 0.9999, T), torch.full((T,), 0.5)):
            _check(ctx, x, u, **WIDE[s])


@pytest.mark.parametrize("V", [1, 2, 64, 1000, 4096, 100_000, 1 << 18])
def test_all_alike(ctx, V):
    T = 9
    u = torch.tensor([0.0, LAST, 0.5, 0.25, 0.1, 0.9, 1 / 3, 2.0**-24, 0.75])
    for value in (0.0, -1e30, 65504.0):
        x = torch.full((T, V), value)
        for s in (dict(), dict(topK=1), dict(topK=V // 2 + 1), dict(topK=V), dict(topP=0.5), dict(topP=0.75, topK=max(1, V // 4)), dict(minP=1.0)):
            _check(ctx, x, u, **s)


@pytest.mark.parametrize("dtype", TYPES)
def test_ties(ctx, dtype):
    """Few different values: cuts and draws fall among equal ones, the first of which come first."""
    g = torch.Generator().manual_seed(1)
    for T, V in ((200, 3000), (9, 70_000)):
        x = torch.randint(-6, 1, (T, V), generator=g).float()
        x[::3, ::2] = -0.0
        u = torch.rand(T, generator=g)
        for s in (dict(), dict(topK=5), dict(topK=431), dict(topK=2999), dict(topP=0.1), dict(topP=0.77), dict(topK=1000, topP=0.63), dict(minP=0.1), dict(minP=0.3, topK=300)):
            _check(ctx, x.to(dtype), u, **s)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [5, 300, 5000, 70_000])
def test_masks(ctx, V, dtype):
    low = torch.finfo(dtype).min
    x, _ = _logits(12, V, torch.float32, V)
    x[0] = -torch.inf
    x[1] = torch.nan
    x[2] = -torch.inf
    x[2, V // 2] = -3.0
    x[3] = torch.nan
    x[3, V - 1] = 2.0
    x[4, ::2] = -torch.inf
    x[5, 1::2] = torch.nan
    x[6] = low
    x[7] = low
    x[7, V // 3] = 1.0
    x[8, V // 2] = torch.inf
    x[9] = -torch.inf
    x[9, 0], x[9, V - 1] = torch.inf, torch.inf
    x[10, 1::2] = -torch.inf
    x[10, 0] = torch.nan
    x[11, 0], x[11, 1] = torch.finfo(dtype).max, low
    for u in (0.0, 0.37, 0.73, LAST):
        for s in (dict(), dict(topK=1), dict(topK=3), dict(topK=200), dict(topP=0.9), dict(topP=0.5, topK=100), dict(minP=0.2), dict(temperature=0.0), dict(temperature=1e-30), dict(temperature=1e30, topP=0.9),
                  dict(topK=V - 1, minP=0.01)):
            _check(ctx, x.to(dtype), torch.full((12,), u), **s)


@pytest.mark.parametrize("V", [70_000, 1 << 18])
def test_rows_that_the_passes_give_up_on(ctx, V):
    x, u = _given_up(V)
    for s in (dict(), dict(topK=20_000), dict(topP=0.4), dict(topP=0.9, minP=0.001), dict(minP=0.0001)):
        _check(ctx, x, u, **s)


def test_smaller_random_numbers_draw_more_likely_items(ctx):
    T = 64
    u = torch.linspace(0, LAST, T)
    for V in (3000, 50_000):
        row = _logits(1, V, torch.float32, V)[0]
        for s in (dict(), dict(topK=50), dict(topP=0.9), dict(minP=0.01)):
            items = _check(ctx, row.expand(T, V).contiguous(), u, **s)
            got = row[0][torch.tensor(items)]
            assert bool((got[1:] <= got[:-1]).all()) and items[0] == int(row[0].argmax())


def test_the_same_items_are_kept_in_either_order(ctx):
    """4096 draws with u spread evenly: each item as often as in the other order, give or take one."""
    k = _kernel(ctx)
    row = torch.randn(300, generator=torch.Generator().manual_seed(5)).cuda()
    n = 4096
    x, u = row.expand(n, 300).contiguous(), ((torch.arange(n) + 0.5) / n).cuda()
    for s in (dict(), dict(topK=25), dict(topP=0.8), dict(minP=0.2), dict(topK=100, topP=0.7, minP=0.05, temperature=0.7)):
        a, b = (torch.bincount(k.sample(x, u, **s, order=order)[0], minlength=300) for order in ("items", "logits"))
        assert int((a - b).abs().max()) <= 2 and torch.equal(a[b > 2] > 0, b[b > 2] > 0)


def test_settings_of_each_row(ctx):
    g = torch.Generator().manual_seed(3)
    T = 400
    pick = lambda v, of: torch.tensor(v, dtype=of)[torch.randint(0, len(v), (T,), generator=g)]  # noqa: E731
    many = dict(temperature=pick([0.0, 0.5, 1.0, 2.0], torch.float32), topK=pick([0, 1, 3, 40, 500, 2500], torch.int32), topP=pick([1.0, 0.5, 0.9, 0.99], torch.float32),
                minP=pick([0.0, 0.01, 0.2], torch.float32))
    for V in (3000, 40_000):
        x, u = _logits(T if V < 10_000 else 60, V, torch.float32, V)
        n = x.shape[0]
        _check(ctx, x, u, **{name: v[:n].clone() for name, v in many.items()})
        for name, v in many.items():
            _check(ctx, x, u, **{name: v[:n].clone()})


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_runs(ctx, dtype):
    k = _kernel(ctx)
    for V in (777, 60_001):
        x, u = _logits(20, V, dtype, V)
        room = torch.full((20, V + 13), torch.nan, dtype=dtype)
        room[:, 5 : 5 + V] = x
        x, room, u = x.cuda(), room.cuda(), u.cuda()
        for s in SETTINGS[:10]:
            a, b, c = (k.sample(y, u, **s, order="logits") for y in (x, room[:, 5 : 5 + V], x))
            assert all(torch.equal(a[i], b[i]) and torch.equal(a[i], c[i]) for i in (0, 1))


@pytest.mark.parametrize("T,V", [(2, 300_000), (40, 60_000), (300, 4000)])
@pytest.mark.parametrize("own", [False, True])
def test_captured(ctx, T, V, own):
    """Two graphs replayed in turn on changed logits, with eager calls of the same context between them; with a workspace each, whatever it
    held before, and without."""
    k = _kernel(ctx)
    x, u = (t.cuda() for t in _logits(T, V, torch.bfloat16, 1))
    settings, graphs, outs = (dict(topP=0.9, temperature=2.0), dict(topK=20, minP=0.01)), [], []
    need = k.workspaceBytes(T, V)
    spaces = [torch.full((need,), 0xAB, dtype=torch.uint8, device="cuda") if own and need else None for _ in settings]
    torch.cuda.synchronize()
    for s, space in zip(settings, spaces):
        items, logs = torch.zeros(T, dtype=torch.int64, device="cuda"), torch.zeros(T, device="cuda")
        k.encode(x, u, items, logs, **s, workspace=space, order="logits")
        ctx.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=ctx.torch_stream()):
            k.encode(x, u, items, logs, **s, workspace=space, order="logits")
        graphs.append(g)
        outs.append((items, logs))
    for i in range(4):
        y, v = _logits(T, V, torch.bfloat16, 10 + i)
        x.copy_(y), u.copy_(v)
        torch.cuda.synchronize()
        want = [k.sample(x, u, **s, order="logits") for s in settings]
        for o in outs:
            o[0].fill_(-7), o[1].fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(ctx.torch_stream()):
            for j in (1, 0, 1) if i % 2 else (0, 1):
                graphs[j].replay()
        k.sample(x, u, topP=0.5, order="logits")
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o[0], w[0]) and bool(((o[1] - w[1]).abs() <= 2e-7 * w[1].abs() + 1e-10).all())


def test_refusals(ctx):
    from vectoraccelerate_amd import VectorError, _lib

    k = _kernel(ctx)
    x, u, items = torch.zeros(4, 50, device="cuda"), torch.zeros(4, device="cuda"), torch.full((4,), 9, device="cuda")
    torch.cuda.synchronize()
    for order in ("", "item", "Logits", None, 1):
        with pytest.raises(VectorError):
            k.encode(x, u, items, order=order)
        with pytest.raises(VectorError):
            k.sample(x, u, order=order)
    for order in (-1, 2):
        d = _lib.SampleDesc(logits=x.data_ptr(), uniforms=u.data_ptr(), stride=50, rows=4, num_items=50, dtype=0, temperature=1.0, top_p=1.0)
        assert ctx.lib.va_sample_in_order(ctx.handle, C.byref(d), order, items.data_ptr(), None) == 1
    assert items.tolist() == [9] * 4


def test_cpp_class(tmp_path):
    """SoftmaxSamplingKernel::sample with an order, run by tests/cpp/va_example."""
    from tests.test_gpu_learning_run import EXE

    if not EXE.exists():
        from vectoraccelerate_amd.build import build_cpp_example

        build_cpp_example()
    Q, N, D, classes = 40, 1500, 32, 8
    g = np.random.default_rng(4)
    for name, n in (("q", Q), ("x", N), ("c", classes)):
        g.standard_normal((n, D), np.float32).tofile(tmp_path / f"{name}.bin")
    proc = subprocess.run([str(EXE), str(tmp_path), str(Q), str(N), str(D), str(classes), "5", "4"], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stderr
    rd = lambda n, kind: np.fromfile(tmp_path / f"{n}.bin", kind)  # noqa: E731
    scores, items, logs = rd("mx_scores", np.float32).reshape(Q, N), rd("falling_items", np.int64), rd("falling_log", np.float32)
    for t in range(Q):
        item, probability, near = drawn(scores[t], 0.375, 1.0, 10, 1.0, 0.0)
        assert near > 2.0**-40 and int(items[t]) == item and abs(float(logs[t]) - np.log(probability)) < 2.0**-22 * abs(np.log(probability)) + 1e-9


def test_without_probabilities_and_far_rows(ctx):
    """No log probabilities asked for; rows more than 2^32 bytes apart."""
    k = _kernel(ctx)
    stride = (1 << 31) + 64
    room = torch.empty(2 * stride + 30_000, dtype=torch.float16, device="cuda")
    for V in (1000, 30_000):
        far = torch.as_strided(room, (3, V), (stride, 1))
        x, u = _logits(3, V, torch.float16, V)
        far.copy_(x)
        dx, du = x.cuda(), u.cuda()
        for s in (dict(), dict(topK=9), dict(topP=0.8, temperature=3.0)):
            a = k.sample(dx, du, **s, order="logits")
            b = k.sample(far, du, **s, order="logits")
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
            items = torch.full((5,), 7, device="cuda")
            torch.cuda.synchronize()
            k.encode(far, du, items[1:4], None, **s, order="logits")
            ctx.synchronize()
            assert items.tolist() == [7, *a[0].tolist(), 7]
    del room, far
    torch.cuda.empty_cache()
