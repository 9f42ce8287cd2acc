"""AdamW over a list of tensors (va_adamw.hip) against 64 bits: sizes around the vector, group and chunk edges, every
combination of types, 32-bit copies, 8-bit moments and their rounding, clipping and skipped steps, steps in a graph."""
from __future__ import annotations

import pytest
import torch

from tests import training_oracle as oracle
from tests.training_oracle import TINY, U, U32

pytestmark = pytest.mark.gpu

F32, F16, BF16, FP8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
KINDS = [(F32, F32, False), (F16, F16, False), (BF16, BF16, False), (F16, F32, False), (BF16, F32, False), (F16, F16, True), (BF16, BF16, True),
         (F16, F32, True), (BF16, F32, True)]
SET = dict(beta1=0.9, beta2=0.99, epsilon=1e-6, weightDecay=0.1)


def _kernel(ctx):
    from vectoraccelerate_amd import AdamWKernel

    return AdamWKernel(ctx)


def _inputs(kernel, sizes, kinds, bits, seed, scale=0.01):
    """Parameters, gradients and a state some steps in."""
    g = torch.Generator().manual_seed(seed)
    normal = lambda n, s: torch.randn(n, generator=g) * s  # noqa: E731
    params = [normal(n, 0.5).to(kinds[i % len(kinds)][0]).cuda() for i, n in enumerate(sizes)]
    grads = [normal(n, scale).to(kinds[i % len(kinds)][1]).cuda() for i, n in enumerate(sizes)]
    state = kernel.state(params, bits)
    masters = [(p.float() + p.float().abs() * U[p.dtype] * 0.4) if kinds[i % len(kinds)][2] else None for i, p in enumerate(params)]
    state.masters = masters if any(k[2] for k in kinds) else None
    for i, n in enumerate(sizes):
        m, r = normal(n, scale), (normal(n, scale).abs() + 0.2 * scale)
        if bits == 32:
            state.first[i].copy_(m)
            state.second[i].copy_(r * r)
        else:
            for x, codes, scales in ((m, state.first[i], state.firstScales[i]), (r, state.second[i], state.secondScales[i])):
                top = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256).amax(1) if n else x
                scales.copy_(top / 448)
                codes.copy_((x / (top / 448).repeat_interleave(256)[:n]).clamp(-448, 448).to(FP8))
    return params, grads, state


def _held(state, i, n, bits):
    """(m, v) of a tensor in 64 bits."""
    m, v = state.first[i].cpu().double().view(-1), state.second[i].cpu().double().view(-1)
    if bits == 8:
        m = m * state.firstScales[i].cpu().double().repeat_interleave(256)[:n]
        v = (v * state.secondScales[i].cpu().double().repeat_interleave(256)[:n]) ** 2
    return m, v


def _like(params, state):
    from vectoraccelerate_amd import AdamWState

    new = lambda l: [torch.full_like(t, 7.0) if t is not None else None for t in l] if l is not None else None  # noqa: E731
    return new(params), AdamWState(*(new(l) for l in (state.first, state.second, state.firstScales, state.secondScales, state.masters)))


def _check(want, got, params, grads, state, out, bits, step, rate, factor=1.0, rates=None, decays=None, beta1=0.9, beta2=0.99, epsilon=1e-6, weightDecay=0.1):
    """A step's results against 64 bits.  Roundings of fp32, u each: the clipping factor 4 and its product 1, the betas and
    their products 2, the sums 1 (8-bit moments: code times scale 1), so m is off by 9 u of its terms' magnitudes and v, whose
    terms are squares of these, by 20 u; its root by 11, the divisor by 15 with the bias correction, the product and the sum."""
    new_params, new_state = out
    for i, p in enumerate(params):
        n = p.numel()
        m0, v0 = _held(state, i, n, bits)
        g = grads[i].cpu().double().view(-1) * factor
        m, v = beta1 * m0 + (1 - beta1) * g, beta2 * v0 + (1 - beta2) * g * g
        em = 9 * U32 * (beta1 * m0.abs() + (1 - beta1) * g.abs()) + 2.0**-148
        r = (rates[i] if rates else 1.0) * rate
        master = state.masters is not None and state.masters[i] is not None
        p0 = (state.masters[i] if master else p).cpu().double().view(-1)
        d = torch.sqrt(v / (1 - beta2**step)) + epsilon
        move = r / (1 - beta1**step) / d
        keep = 1 - r * weightDecay * (decays[i] if decays else 1.0)
        p1 = p0 * keep - move * m
        ep = move * (em + 20 * U32 * m.abs()) + 3 * U32 * p0.abs() + U32 * p1.abs()
        if master:
            oracle.close(new_state.masters[i].view(-1), p1, ep, f"master {i}")
            assert torch.equal(new_params[i], new_state.masters[i].view_as(new_params[i]).to(p.dtype)), f"parameter {i}"
        else:
            oracle.close(new_params[i].view(-1), p1, ep + (U[p.dtype] if p.dtype != F32 else 0) * (p1.abs() + ep) + TINY[p.dtype], f"parameter {i}")
        if bits == 32:
            oracle.close(new_state.first[i], m, em, f"first {i}")
            oracle.close(new_state.second[i], v, 20 * U32 * v + 2.0**-148, f"second {i}")
            continue
        for name, x, ex, scales, codes in (("first", m, em, new_state.firstScales[i], new_state.first[i]),
                                           ("second", v.sqrt(), 11 * U32 * v.sqrt(), new_state.secondScales[i], new_state.second[i])):
            pad = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256)
            epad = torch.nn.functional.pad(ex, (0, -n % 256)).view(-1, 256).amax(1)
            oracle.close(scales, pad.amax(1) / 448, epad / 448 + 2 * U32 * pad.amax(1) / 448, f"{name} scales {i}")
            s = scales.cpu().double().repeat_interleave(256)[:n]
            # e4m3 has eight values in each binary order from 2^-6 on, and steps of 2^-9 below: less than one step off (near
            # a power of two the next order's)
            z = (x.abs() / s).clamp(max=448.0) * (1 + 2.0**-12)
            width = torch.exp2((torch.frexp(z).exponent - 1).clamp(min=-6).double() - 3)
            width = torch.where((name == "second") & (z < 2.0**-9), 2.0**-9, width)
            oracle.close(codes.cpu().double() * s, x, width * s * (1 + 8 * U32) + ex + 4 * U32 * x.abs(), f"{name} codes {i}")
            if name == "second":
                assert (codes.cpu().float()[x > 0] > 0).all()


def _step(ctx, params, grads, state, bits, in_place=False, step=7, rate=0.02, factor=1.0, rates=None, decays=None, **more):
    k = _kernel(ctx)
    before = [t.clone() for t in params], _copy(state)
    out = (params, state) if in_place else _like(params, state)
    lst = k.tensorList(params, grads, state, None if in_place else out, rates, decays)
    k.step(lst, step, rate, **SET, **more)
    _check(None, None, before[0], grads, before[1], out, bits, step, rate, factor, rates, decays)
    if not in_place:  # what is read stays as it was
        assert all(torch.equal(a, b) for a, b in zip(params, before[0]))
    return out


def _copy(state):
    from vectoraccelerate_amd import AdamWState

    c = lambda l: [t.clone() if t is not None else None for t in l] if l is not None else None  # noqa: E731
    return AdamWState(*(c(l) for l in (state.first, state.second, state.firstScales, state.secondScales, state.masters)))


def _all(out):
    p, s = out
    return [t for l in (p, s.first, s.second, s.firstScales, s.secondScales, s.masters) if l is not None for t in l if t is not None]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("in_place", [False, True])
def test_types(ctx, kind, bits, in_place):
    k = _kernel(ctx)
    _step(ctx, *_inputs(k, [5003, 256, 17], [kind], bits, 1), bits, in_place)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 7, 8, 9, 255, 256, 257, 511, 1023, 1024, 1025, 2047, 2048, 2049, 4097, 100_003, 1_000_001])
def test_sizes(ctx, n, bits):
    k = _kernel(ctx)
    _step(ctx, *_inputs(k, [n], [KINDS[n % 9]], bits, n), bits)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [2, 63, 64, 65, 129, 400])
def test_lists(ctx, count, bits):
    g = torch.Generator().manual_seed(count)
    sizes = torch.randint(0, 5000, (count,), generator=g).tolist()
    sizes[0], sizes[count // 2], sizes[-1] = 0, 300_000, 0
    rates = (torch.rand(count, generator=g) * 2).tolist()
    decays = [float(i % 2) for i in range(count)]
    rates = [float(torch.tensor(r, dtype=F32)) for r in rates]
    k = _kernel(ctx)
    # (copies for some of the tensors alone)
    _step(ctx, *_inputs(k, sizes, KINDS, bits, count), bits, count % 2 == 0, rates=rates, decays=decays)


@pytest.mark.parametrize("bits", [32, 8])
def test_views_at_any_offset(ctx, bits):
    k = _kernel(ctx)
    params, grads, state = _inputs(k, [3001, 777, 4096], [(BF16, BF16, True), (F32, F32, False), (F16, F32, True)], bits, 4)

    def shifted(t, by):
        if t is None:
            return None
        room = torch.zeros(t.numel() + 16, dtype=t.dtype, device="cuda")
        room[by : by + t.numel()] = t
        return room[by : by + t.numel()]

    from vectoraccelerate_amd import AdamWState

    move = lambda l, by: [shifted(t, by + i) for i, t in enumerate(l)] if l is not None else None  # noqa: E731
    moved = AdamWState(*(move(l, 1 + j) for j, l in enumerate((state.first, state.second, state.firstScales, state.secondScales, state.masters))))
    a = _step(ctx, params, grads, state, bits)
    b = _step(ctx, move(params, 3), move(grads, 1), moved, bits, True)
    assert all(torch.equal(x, y) for x, y in zip(_all(a), _all(b)))


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping(ctx, bits):
    """The factor of a given norm and of gradScale; a norm below the bound changes nothing."""
    k = _kernel(ctx)
    args = _inputs(k, [3000, 12_345], [(BF16, BF16, False)], bits, 5)
    norm = torch.tensor([3.0], device="cuda")
    _step(ctx, *args, bits, gradNorm=norm, maxNorm=0.75, factor=0.75 / (3.0 + 1e-6))
    _step(ctx, *args, bits, gradNorm=norm, maxNorm=4.0)
    _step(ctx, *args, bits, gradNorm=norm, maxNorm=0.75, gradScale=0.5, factor=0.5 * 0.75 / (1.5 + 1e-6))
    _step(ctx, *args, bits, gradScale=0.125, factor=0.125)
    _step(ctx, *args, bits, gradNorm=norm, maxNorm=0.0, factor=0.0)
    _step(ctx, *args, bits, gradNorm=norm)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("value", [float("inf"), float("nan"), -float("inf")])
def test_a_norm_that_is_not_finite_skips_the_step(ctx, bits, value):
    k = _kernel(ctx)
    params, grads, state = _inputs(k, [1, 3000, 256, 2048, 5], KINDS[3:8], bits, 6)
    grads[1][7] = value
    norm = torch.tensor([value], device="cuda")
    want = [t.clone() for t in _all((params, state))]
    out = _like(params, state)
    k.step(k.tensorList(params, grads, state, out), 3, 0.1, gradNorm=norm, maxNorm=1.0)
    k.step(k.tensorList(params, grads, state), 3, 0.1, gradNorm=norm)
    for got in (_all(out), _all((params, state))):
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(want, got))


def test_a_value_that_is_not_finite_stays_its_own(ctx):
    """32 bits: its own value alone; 8 bits: its group."""
    k = _kernel(ctx)
    for bits in (32, 8):
        params, grads, state = _inputs(k, [1000, 700], [KINDS[0]], bits, 8)
        clean = _like(params, state)
        k.step(k.tensorList(params, grads, state, clean), 2, 0.1)
        for bad in (float("nan"), float("inf")):
            g = [x.clone() for x in grads]
            g[0][300] = bad
            out = _like(params, state)
            k.step(k.tensorList(params, g, state, out), 2, 0.1)
            off = out[0][0] != clean[0][0]
            assert int(off.sum()) == 1 and bool(off[300]) and torch.equal(out[0][1], clean[0][1])
            if bits == 8:
                same = torch.arange(4, device="cuda") != 1  # 300 lies in the second group
                for a, b in ((out[1].firstScales[0], clean[1].firstScales[0]), (out[1].secondScales[0], clean[1].secondScales[0])):
                    assert not torch.isfinite(a[1]) and torch.equal(a[same], b[same])
                assert torch.equal(out[1].first[0][512:].float(), clean[1].first[0][512:].float())


def _emulated(x, seed, step, least):
    """Codes and scales of fp32 values whose place in the list is their index, in ordinary torch operations; which: 0 first, 1 second."""
    mask = (1 << 64) - 1

    def mixed(z):
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & mask
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & mask
        return z ^ (z >> 31)

    golden = 0x9E3779B97F4A7C15
    base = mixed((seed + golden * step) & mask)
    random = []
    for j in range(-(-x.numel() // 2)):
        z = mixed((base + golden * (j + 1)) & mask)
        random += [(z >> (16 * least)) & 0xFFFF, (z >> (32 + 16 * least)) & 0xFFFF]
    random = torch.tensor(random[: x.numel()], dtype=F32)
    n = x.numel()
    top = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256).amax(1)
    t = top.repeat_interleave(256)[:n]
    z = (x.abs() * (torch.tensor(448.0) / t)).clamp(max=448.0)
    width = torch.exp2((torch.frexp(z).exponent - 1).clamp(min=-6).float() - 3)
    z = (torch.floor(z / width + random / 65536) * width).clamp(max=448.0)
    if least:
        z = torch.where((x > 0) & (z == 0), 2.0**-9, z)
    return torch.copysign(z, x).to(FP8), top / 448.0


@pytest.mark.parametrize("seed,step", [(0, 1), (12345678901234567890, 77), (2**64 - 1, 10**6)])
def test_rounding_of_8_bits(ctx, seed, step):
    """With betas of 0 the moments are the gradient and its magnitude: every code is known."""
    k = _kernel(ctx)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3001, generator=g) * torch.exp2(torch.randint(-22, 1, (3001,), generator=g).float())
    x[600:620] = 0.0
    p, grad = torch.zeros(3001, device="cuda"), x.cuda()
    state = k.state([p], 8)
    k.step(k.tensorList([p], [grad], state), step, 0.1, beta1=0.0, beta2=0.0, seed=seed)
    for least, values, codes, scales in ((0, x, state.first[0], state.firstScales[0]), (1, (x * x).sqrt(), state.second[0], state.secondScales[0])):
        want, s = _emulated(values, seed, step, least)
        assert torch.equal(codes.cpu().view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales.cpu(), s)


def test_rounding_is_right_on_average(ctx):
    """A moment between two codes is the upper one as often as it has to be: over N values the mean is off by less than
    6 sigma of N independent choices, half a code's width each at most; another seed chooses anew."""
    k = _kernel(ctx)
    n = 1 << 20
    g = torch.full((n,), 0.3, device="cuda")
    g[::256] = 1.0  # each group's largest: 0.3 is 134.4 of 448, between 128 and 144
    p = torch.zeros(n, device="cuda")
    got = []
    for seed in (1, 2):
        state = k.state([p], 8)
        k.step(k.tensorList([p], [g], state, ([torch.empty_like(p)], state)), 1, 0.0, beta1=0.0, beta2=0.0, seed=seed)
        for codes in (state.first[0], state.second[0]):
            c = codes.float()[torch.arange(n, device="cuda") % 256 != 0]
            assert set(c.unique().tolist()) == {128.0, 144.0}
            assert abs(float(c.double().mean()) - 134.4) < 6 * 8 / c.numel() ** 0.5 + 1e-4
            got.append(c)
    for a in range(4):
        for b in range(a):
            # two independent choices agree with 0.6^2 + 0.4^2 = 0.52
            assert abs(float((got[a] == got[b]).double().mean()) - 0.52) < 0.01


def test_a_moment_in_8_bits_comes_down(ctx):
    """With no more gradients v falls by beta2 a step on average, though a step is a hundredth of a code's width.  r = 0.42 of
    its group's largest falls to 0.42 beta2^(t/2) of the same largest (whose gradients go on).  A step's choice between two codes a
    width w <= r / 8 apart has at most the variance (the move) w = 0.001 r r / 8; 200 of them 0.025 r^2; of the mean of 4080 values
    6 sigma are 0.015 r."""
    k = _kernel(ctx)
    n = 16 * 256
    p = torch.zeros(n, device="cuda")
    g = torch.full((n,), 0.42, device="cuda")
    g[::256] = 1.0
    state = k.state([p], 8)
    lst = k.tensorList([p], [g], state)
    k.step(lst, 1, 0.0, beta1=0.0, beta2=0.0)
    rest = torch.arange(n, device="cuda") % 256 != 0
    r0 = (state.second[0].float() * state.secondScales[0].repeat_interleave(256))[rest].double().mean()
    g[rest] = 0.0
    for t in range(200):
        k.encode(lst, 2 + t, 0.0, beta2=0.998)
    ctx.synchronize()
    r = (state.second[0].float() * state.secondScales[0].repeat_interleave(256))[rest].double().mean()
    assert abs(float(r / r0) / 0.998**100 - 1) < 0.015


def test_zeros_and_tiny_values(ctx):
    k = _kernel(ctx)
    p = torch.ones(1024, device="cuda")
    g = torch.zeros(1024, device="cuda")
    g[256:512] = 1e-35  # below 2^-100
    state = k.state([p], 8)
    k.step(k.tensorList([p], [g], state), 1, 0.5, weightDecay=0.0)
    assert bool((p[:256] == 1).all() and (p[512:] == 1).all())
    assert (state.first[0].float() == 0).all() and (state.firstScales[0] == 0).all() and (state.secondScales[0] == 0).all()
    k.step(k.tensorList([p], [g], state), 2, 0.5, weightDecay=0.0)
    assert torch.isfinite(p).all()


@pytest.mark.parametrize("steps", [25])
def test_steps_follow_another_implementation(ctx, steps):
    """25 steps beside torch's optimiser in 64 bits.  A step adds at most 40 u of its move (a few of the rate: the moments' own
    errors fade with the betas, 1 / (1 - beta1) = 10 steps of 9 u) and 4 u of the value."""
    k = _kernel(ctx)
    g = torch.Generator().manual_seed(0)
    sizes = [1000, 37]
    start = [torch.randn(n, generator=g) for n in sizes]
    ref = [torch.nn.Parameter(p.double()) for p in start]
    opt = torch.optim.AdamW(ref, lr=0.01, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
    p = [s.cuda() for s in start]
    grads = [torch.zeros_like(x) for x in p]
    lst = k.tensorList(p, grads, k.state(p))
    for t in range(1, steps + 1):
        for i, n in enumerate(sizes):
            d = torch.randn(n, generator=g) * (1 + i)
            grads[i].copy_(d)
            ref[i].grad = d.double()
        opt.step()
        k.step(lst, t, 0.01, **SET)
    for a, b in zip(p, ref):
        b = b.detach()
        oracle.close(a, b, steps * (4 * U32 * (b.abs() + 0.3) + 0.01 * 10 * 130 * U32), "parameters")


def test_step_and_rate_on_the_device(ctx):
    k = _kernel(ctx)
    for bits in (32, 8):
        params, grads, state = _inputs(k, [3000, 5], [KINDS[2]], bits, 11)
        a, b = _like(params, state), _like(params, state)
        k.step(k.tensorList(params, grads, state, a), 9, 0.25, seed=4)
        k.step(k.tensorList(params, grads, state, b), torch.tensor([9], device="cuda"), torch.tensor([0.25], device="cuda"), seed=4)
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(_all(a), _all(b)))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(ctx, bits):
    """Two graphs (a step, and a step with clipping by a norm computed before it) replayed in turn with eager steps between
    them go through the same values as eager steps alone."""
    from vectoraccelerate_amd import GradientClipKernel

    k, clip = _kernel(ctx), GradientClipKernel(ctx)
    params, grads, state = _inputs(k, [5000, 300], [(BF16, BF16, True)], bits, 12)
    first = _copy(state), [p.clone() for p in params]
    t, rate, norm = torch.tensor([1], device="cuda"), torch.tensor([0.01], device="cuda"), torch.zeros(1, device="cuda")
    lst = k.tensorList(params, grads, state)
    gl = clip.tensorList(grads)
    clip.encode(gl, float("inf"), norm)  # (the scratch arena has its size before the capture)
    ctx.synchronize()

    def one():
        k.encode(lst, t, rate, seed=1, **SET)
        with torch.cuda.stream(ctx.torch_stream()):
            t.add_(1)

    def two():
        clip.encode(gl, float("inf"), norm)
        k.encode(lst, t, rate, seed=2, gradNorm=norm, maxNorm=0.01, **SET)
        with torch.cuda.stream(ctx.torch_stream()):
            t.add_(1)

    def start():
        torch.cuda.synchronize()
        for a, b in zip(_all((params, state)), _all((first[1], first[0]))):
            a.copy_(b)
        t.fill_(1)
        torch.cuda.synchronize()

    torch.cuda.synchronize()
    order = [0, 1, 0, 0, 1, 1, 0]
    for i in order:
        (one, two)[i]()
    ctx.synchronize()
    want = [x.clone() for x in _all((params, state))]
    graphs = []
    for f in (one, two):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=ctx.torch_stream()):
            f()
        graphs.append(g)
    for _ in range(3):
        start()
        for j, i in enumerate(order):
            with torch.cuda.stream(ctx.torch_stream()):
                graphs[i].replay() if j % 3 else (one, two)[i]()
            if j == 2:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(want, _all((params, state))))


@pytest.mark.parametrize("bits", [32, 8])
def test_runs_agree_bit_for_bit(ctx, bits):
    k = _kernel(ctx)
    args = _inputs(k, [100_000, 3, 70_001] * 20, KINDS, bits, 9)
    a, b = (_like(args[0], args[2]) for _ in range(2))
    for out in (a, b):
        k.step(k.tensorList(*args, out), 5, 0.01, seed=3)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(_all(a), _all(b)))


def test_more_than_32_bits_of_values(ctx):
    """The last values of a tensor of 2^32 + 300, in 8 bits."""
    k = _kernel(ctx)
    n = (1 << 32) + 300
    p, g = torch.zeros(n, dtype=BF16, device="cuda"), torch.zeros(n, dtype=BF16, device="cuda")
    state = k.state([p], 8)
    p[-500:] = 1.0
    g[-500:] = torch.linspace(-1, 1, 500, device="cuda").to(BF16)
    k.step(k.tensorList([p], [g], state), 1, 0.5, weightDecay=0.0, seed=1)
    want = 1.0 - 0.5 * torch.sign(g[-500:].float())
    # (v = 0.001 g^2 and m = 0.1 g, corrected: the move is the rate, but for epsilon and the betas' rounding)
    far = g[-500:].float().abs() > 1e-3
    assert float((p[-500:].float() - want)[far].abs().max()) < 2**-7
    assert int((p[:-500] != 0).sum()) == 0
    assert float(state.firstScales[0][-1]) > 0 and float(state.firstScales[0][-4:].min()) >= 0 and int((state.firstScales[0] != 0).sum()) == 3
    del p, g, state
    torch.cuda.empty_cache()


def test_another_stream(ctx):
    """A context on a torch stream: the step is ordered by that stream alone."""
    import ctypes as C

    from vectoraccelerate_amd import AdamWKernel, GPUContext

    stream = torch.cuda.Stream()
    c = GPUContext(0)
    h = C.c_void_p()
    c.check(c.lib.va_context_create_with_stream(0, C.c_void_p(stream.cuda_stream), C.byref(h)), "create")
    c.close()
    c._h, c._ext_stream = h, None
    k = AdamWKernel(c)
    p, g = torch.ones(100_000, device="cuda"), torch.zeros(100_000, device="cuda")
    lst = k.tensorList([p], [g], k.state([p]))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        slow = torch.randn(3000, 3000, device="cuda")
        for _ in range(8):
            slow = slow @ slow * 1e-2
        g.copy_(torch.where(torch.isnan(slow.view(-1)[:100_000]), 1.0, 1.0))
        k.encode(lst, 1, 0.5, weightDecay=0.0)
        q = p * 1.0
    stream.synchronize()
    assert float((q - 0.5).abs().max()) < 1e-5
    lst.close()
    c.close()


def test_refusals(ctx):
    from vectoraccelerate_amd import AdamWState, VectorError

    k = _kernel(ctx)
    p, g = torch.ones(600, device="cuda"), torch.ones(600, device="cuda")
    s, s8 = k.state([p]), k.state([p], 8)
    lst = k.tensorList([p], [g], s)
    room = torch.zeros(1200, device="cuda")
    norm = torch.ones(1, device="cuda")
    bf = p.bfloat16()
    for f in (lambda: k.tensorList([p], [], s), lambda: k.tensorList([p], [g[:5]], s), lambda: k.tensorList([p], [g.half()], s), lambda: k.tensorList([p.double()], [g], s),
              lambda: k.tensorList([p.cpu()], [g], s), lambda: k.tensorList([p], [g.cpu()], s), lambda: k.tensorList([p, p], [g, g], k.state([p, p])),
              lambda: k.tensorList([p], [p], s), lambda: k.tensorList([room[:600], room[300:900]], [g, g], k.state([p, p])),
              lambda: k.tensorList([room[:600]], [g], s, ([room[300:900]], s)), lambda: k.tensorList([p], [s.first[0]], s),
              lambda: k.tensorList([p], [g], AdamWState(s.first, s.first)), lambda: k.tensorList([p], [g], AdamWState(s8.first, s8.second)),
              lambda: k.tensorList([p], [g], AdamWState(s.first, s.second, s8.firstScales, s8.secondScales)),
              lambda: k.tensorList([p], [g], AdamWState(s8.first, s8.second, s8.firstScales, None)),
              lambda: k.tensorList([p], [g], AdamWState(s8.first, s8.second, [norm], s8.secondScales)),
              lambda: k.tensorList([p], [g], AdamWState(s.first, s.second, masters=[room[:600]])),
              lambda: k.tensorList([p], [g], s, ([room[:600]], s8)), lambda: k.tensorList([p], [g], s, ([], s)),
              lambda: k.tensorList([bf], [g], AdamWState(s.first, s.second, masters=[room[:600]]), ([bf], AdamWState(s.first, s.second, masters=[None]))),
              lambda: k.tensorList([p], [g], s, rateFactors=[-1.0]), lambda: k.tensorList([p], [g], s, decayFactors=[float("nan")]),
              lambda: k.tensorList([p], [g], s, rateFactors=[1.0, 1.0]), lambda: k.state([p], 16), lambda: k.encode(lst, 0, 0.1), lambda: k.encode(lst, 1, -0.1),
              lambda: k.encode(lst, 1, float("nan")), lambda: k.encode(lst, 1, 0.1, beta1=1.0), lambda: k.encode(lst, 1, 0.1, beta2=-0.1),
              lambda: k.encode(lst, 1, 0.1, epsilon=-1.0), lambda: k.encode(lst, 1, 0.1, weightDecay=float("inf")), lambda: k.encode(lst, 1, 0.1, maxNorm=1.0),
              lambda: k.encode(lst, 1, 0.1, gradNorm=norm, maxNorm=-1.0), lambda: k.encode(lst, 1, 0.1, gradNorm=norm.half(), maxNorm=1.0),
              lambda: k.encode(lst, 1, 0.1, gradScale=-1.0), lambda: k.encode(lst, torch.ones(1, device="cuda"), 0.1),
              lambda: k.encode(lst, 1, torch.ones(1, device="cuda").double())):
        with pytest.raises(VectorError):
            f()
    assert (p == 1).all()
    # a gradient may be shared; empty lists and tensors are nothing to do
    q = torch.ones(600, device="cuda")
    k.step(k.tensorList([p, q], [g, g], k.state([p, q])), 1, 0.1)
    assert torch.equal(p, q) and not torch.equal(p, g)
    k.step(k.tensorList([], [], k.state([])), 1, 0.1)
    e = torch.empty(0, device="cuda")
    k.step(k.tensorList([e], [e], k.state([e])), 1, 0.1)
    lst.close()
    with pytest.raises(VectorError):
        k.encode(lst, 1, 0.1)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("kind", [0, 2, 6])
def test_the_least_epsilons(ctx, bits, kind):
    """Divisors below fp32's normal values: epsilon alone, where v is zero; and m = v = 0, which moves nothing."""
    k = _kernel(ctx)
    n, rate, step = 700, 1e-3, 3
    for epsilon in (1e-45, 1e-40, 1.1754e-38, 1.2e-38, 1e-30, 1e30, 2e30, 3e38):
        p = [torch.randn(n, generator=torch.Generator().manual_seed(1)).to(KINDS[kind][0]).cuda()]
        g = [torch.zeros(n, dtype=KINDS[kind][1], device="cuda")]
        state = k.state(p, bits, masters=KINDS[kind][2])
        if bits == 32:
            state.first[0][::2] = 1e-37
        out = _like(p, state)
        k.step(k.tensorList(p, g, state, outputs=out), step, rate, beta1=0.9, beta2=0.99, epsilon=epsilon, weightDecay=0.0)
        m = 0.9 * state.first[0].cpu().double() if bits == 32 else torch.zeros(n, dtype=torch.float64)
        eps = float(torch.tensor(epsilon, dtype=F32))  # (what the step has of it)
        want = (state.masters[0] if KINDS[kind][2] else p[0]).cpu().double().view(-1) - rate / (1 - 0.9**step) * m / eps
        got = out[0][0].cpu().double()
        assert bool(torch.isfinite(got).all())
        # m is off by a half of the least fp32 value and 3 u, the quotient and the product by an u each, the sum by its own rounding
        loose = (5 * U32 * m.abs() + 2.0**-149) * (rate / (1 - 0.9**step) / eps) + 2 * U32 * want.abs() + U[p[0].dtype] * want.abs() + TINY[p[0].dtype]
        assert bool(((got - want).abs() <= loose).all()), f"epsilon {epsilon}"
        assert torch.equal(got[1::2], p[0].cpu().double()[1::2])
