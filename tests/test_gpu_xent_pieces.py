"""Softmax cross entropy over more items than one piece of the workspaces holds, value by value: the loss, every
hidden gradient, and the items' gradients around the pieces' edges (the definition in 64 bits, on the device)."""
from __future__ import annotations

import pytest
import torch

from tests.training_oracle import TINY, U, U32

pytestmark = pytest.mark.gpu

COPIES, DL = 256 << 20, 512 << 20  # bytes of copied items and of dl that a piece holds


def _piece(T, V, D, dtype, copied):
    """Items of a piece of the backward pass, and of the forward pass where its items are copied."""
    size = 4 if dtype == torch.float32 else 2
    row = -(-D * size // 128) * 128
    forward = COPIES // row // 256 * 256
    backward = DL // (T * size) // 256 * 256
    return forward, min(forward, backward) if copied else backward


def _near(got, want, bound, name):
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN elsewhere"
    off = (got.double() - want).abs() > bound
    assert not bool(off.any()), f"{name}: {int(off.sum())} of {off.numel()} off"


# (rows, items, dimensions, type, whether the items are copied): fp32 planes, fp32 as it is, odd rows, rows in place
CASES = [
    (100, 400_003, 384, torch.float32, True),
    (70, 2 * 174_592 + 70, 384, torch.float32, True),  # the last piece has fewer stages than dh has shares
    (20, 400_003, 384, torch.float32, True),
    (64, 300_001, 513, torch.bfloat16, True),
    (9, 2 * 232_960 + 1, 513, torch.float16, True),
    (300, 300_001, 512, torch.bfloat16, True),
    (4100, 70_001, 64, torch.bfloat16, False),
    (2100, 140_000, 40, torch.float32, True),
]


@pytest.mark.parametrize("T,V,D,dtype,copied", CASES)
@pytest.mark.parametrize("masks", [False, True])
def test_pieces(ctx, T, V, D, dtype, copied, masks):
    """With masks: corrections, and deleted items that hold NaN in the last piece alone."""
    from vectoraccelerate_amd import SoftmaxCrossEntropyKernel

    g = torch.Generator("cuda").manual_seed(T + V)
    scale = 12.0
    h, w = torch.randn(T, D, device="cuda", generator=g), torch.randn(V, D, device="cuda", generator=g)
    h, w = (h / h.norm(dim=1, keepdim=True)).to(dtype), (w / w.norm(dim=1, keepdim=True)).to(dtype)
    forward, piece = _piece(T, V, D, dtype, copied or masks)
    assert V > piece, "more than one piece"
    edges = sorted({e for p in (forward, piece) for c in range(0, V, p) for e in (c - 1, c, c + 1, c + p - 1) if 0 <= e < V} | {V - 2, V - 1})
    y = torch.randint(0, V, (T,), device="cuda", generator=g)
    n = min(T, len(edges))
    y[:n] = torch.tensor(edges[-n:], device="cuda")
    y[T // 2] = -100
    off = None
    if masks:
        off = -torch.log1p(torch.rand(V, device="cuda", generator=g) * 8.0)
        dead = torch.rand(V, device="cuda", generator=g) < 0.05
        dead[y.clamp(min=0)] = False
        off[dead] = -torch.inf
        last = dead.clone()
        last[: (V - 1) // piece * piece] = False
        w[last] = torch.nan
    k = SoftmaxCrossEntropyKernel(ctx)
    res = k.forward(h, w, y, "sum", scale, off)
    gh, gw = k.backward(h, w, y, res.logSumExp, None, "sum", scale, off)

    H, W = h.double(), w.double()
    if masks:
        W[dead] = 0.0
    # bounds as in the small tests: the logits' products and sum, the sum of the exponentials, dl's rounding
    full = dtype == torch.float32
    z = scale * (H @ W.T)
    if masks:
        z += off.double()
    ez = scale * ((D + 4) * U32 + (2.0**-20 if full else 0.0)) * (H.abs() @ W.abs().T)
    ez += 4 * U32 * (z.abs().nan_to_num(posinf=0.0) + (off.double().abs().nan_to_num(posinf=0.0) if masks else 0.0))
    if full:
        ez += scale * D * 2.0**-38 * H.abs().amax(1)[:, None] * W.abs().amax(1)[None, :]
    lse = torch.logsumexp(z, 1)
    top = ez.amax(1)
    e_lse = top + 2.0**-16 + 4 * U32 * lse.abs()
    at = y.clamp(min=0)
    ly = z.gather(1, at[:, None]).squeeze(1)
    counted = y >= 0
    loss = torch.where(counted, lse - ly, 0.0)
    e_loss = top + e_lse + 4 * U32 * ly.abs()
    _near(res.logSumExp, lse, e_lse, "lse")
    _near(res.loss, loss, e_loss, "loss")
    _near(res.reduced, loss.sum().view(1), (e_loss[counted].sum() + 2 * U32 * loss.sum().abs()).view(1), "sum")
    p = torch.exp(z - lse[:, None]) * counted[:, None]
    del z
    edl = p * (ez + e_lse[:, None]) + 2.0**-126
    del ez
    p[torch.nonzero(counted).squeeze(1), y[counted]] -= 1.0  # dl
    edl += p.abs() * ((0 if full else U[dtype]) + 4 * U32) + (2.0**-38 if dtype == torch.float16 else 0.0)
    sums = (V + 8) * U32 if full else 2.0**-16
    want = scale * (p @ W)
    _near(gh, want, scale * (edl @ W.abs()) + sums * scale * (p.abs() @ W.abs()) + 2 * U[dtype] * want.abs() + TINY[dtype], "grad_hidden")
    around = sorted({j for e in edges for j in range(max(0, e - 40), min(V, e + 40))})
    rest = torch.randint(0, V, (2000,), generator=torch.Generator().manual_seed(1)).tolist()
    some = torch.tensor(sorted(set(around + rest)), device="cuda")
    want = scale * (p[:, some].T @ H)
    mag = p[:, some].abs().T @ H.abs()
    _near(gw[some], want, scale * (edl[:, some].T @ H.abs()) + (T + 8) * U32 * scale * mag + 2 * U[dtype] * want.abs() + TINY[dtype], "grad_items")
    assert not bool(torch.isnan(gw).any())
    if masks:
        assert bool((gw[dead] == 0).all())
