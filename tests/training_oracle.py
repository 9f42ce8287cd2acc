"""Plain 64-bit forms of the training and serving operators, and the error bounds their tests use.

Everything is computed on the CPU in float64 from the inputs as the kernels get them (already rounded
to their type).  A bound is the sum of what each rounding may contribute, derived next to it; u is the
unit roundoff of a type (2^-24, 2^-11, 2^-8 for round to nearest: half an ulp is at most u |x|).
"""
from __future__ import annotations

import torch

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
# the smallest step of a type (half of it is the largest error of a subnormal result)
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}
U32 = 2.0**-24


def xent(hidden, items, targets, scale, offsets, ignore, grad):
    """loss, lse, dl-based gradients and their bounds, for row gradients `grad` [T] (float64).

    logits: each product of two 16-bit values is exact in fp32 and D of them are added: (D + 2) u32 of
    the sum of magnitudes.  fp32 values are two fp16 planes each: a value is off by 2^-22 of itself (a
    residue below 2^-11 rounded to 11 bits), or, far below its row's largest, by 2^-39 of that; the
    product of the two residues (2^-22) is left out; 2^-20 of the magnitudes covers the three.
    """
    dtype = hidden.dtype
    h, w = hidden.cpu().double(), items.cpu().double()
    T, V = h.shape[0], w.shape[0]
    D = h.shape[1]
    off = offsets.cpu().double() if offsets is not None else torch.zeros(V, dtype=torch.float64)
    masked = torch.isneginf(off)
    w = torch.where(masked[:, None], 0.0, w)
    tg = targets.cpu()
    none = tg == ignore
    valid = (tg >= 0) & (tg < V) & ~none
    hz = torch.where(valid[:, None], h, 0.0)
    z = scale * (h @ w.T) + off
    z[:, masked] = -torch.inf
    mag = abs(scale) * (h.abs() @ w.abs().T)
    per = (D + 4) * U32 + (2.0**-20 if dtype == torch.float32 else 0.0)
    # + the product with the scale, the addition of the offset, and its logarithm's base change (2 u32 |z|)
    ez = per * mag + 4 * U32 * (z.abs().nan_to_num(posinf=0.0, neginf=0.0) + off.abs().nan_to_num(posinf=0.0, neginf=0.0))
    lse = torch.logsumexp(z, 1)
    empty = torch.isneginf(lse)
    at = tg.clamp(0, V - 1)
    ly = z.gather(1, at[:, None]).squeeze(1)
    loss = torch.where(none, 0.0, torch.where(empty, 0.0, torch.where(valid, lse - ly, torch.nan)))
    # lse moves by at most the largest logit error; V positive terms are added in fp32 trees of at most 2^7
    # consecutive terms (2^-17), exp2 and log are good to 2 u32; then u32 of lse itself
    top = ez.max(1).values
    elog = 2.0**-16
    e_lse = top + elog + 4 * U32 * lse.abs().nan_to_num(posinf=0.0, neginf=0.0)
    e_loss = 2 * top + elog + 4 * U32 * ly.abs().nan_to_num(posinf=0.0, neginf=0.0)
    p = torch.exp(z - torch.where(empty, 0.0, lse)[:, None])
    p[empty] = 0.0
    hit = valid & ~empty & ~masked[at]
    y = torch.zeros_like(p)
    y[hit, at[hit]] = 1.0
    g = torch.where(valid & ~empty, grad.double().cpu(), 0.0)[:, None]
    dl = torch.where(g == 0.0, 0.0, (p - y) * g)
    # dl: p is off by p (its logit's and lse's errors), rounded to the type (fp32: two planes, 2^-22)
    u = U[dtype] if dtype != torch.float32 else 2.0**-21
    edl = g.abs() * p * (ez + e_lse[:, None]) + dl.abs() * (u + 4 * U32) + g.abs().max() * 2.0**-38
    sums = (T + V + 8) * U32 if dtype == torch.float32 else 2.0**-16
    more = 2.0**-20 if dtype == torch.float32 else 0.0  # the planes of the other operand and the missing product
    gh, gw = scale * (dl @ w), scale * (dl.T @ hz)
    s = abs(scale)
    e_gh = s * (edl @ w.abs()) + (sums + more) * s * (dl.abs() @ w.abs()) + 2 * U[dtype] * gh.abs() + TINY[dtype]
    e_gw = s * (edl.T @ hz.abs()) + (sums + more) * s * (dl.abs().T @ hz.abs()) + 2 * U[dtype] * gw.abs() + TINY[dtype]
    return {"loss": (loss, e_loss), "lse": (lse, e_lse), "grad_hidden": (gh, e_gh), "grad_items": (gw, e_gw)}


def close(got, want, bound, name):
    """Finite values within the bound; the others alike."""
    got = got.detach().cpu().double()
    want = want.broadcast_to(got.shape)
    bound = bound.broadcast_to(got.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN elsewhere"
    other = ~fine & ~torch.isnan(want)
    assert torch.equal(got[other], want[other]), f"{name}: infinities differ"
    d = (got[fine] - want[fine]).abs()
    b = bound[fine]
    bad = d > b
    if bool(bad.any()):
        i = int((d / b.clamp(min=1e-300)).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {d.numel()} off, worst {float(d[i])} where {float(b[i])} is allowed "
                             f"(value {float(want[fine][i])})")


def rms(x, residual, weight, eps):
    """r, inverse rms, y, and the relative error bound of y before its own rounding: the sum of D squares in
    a lane's chain of at most 32 and a tree, (48 u32), half of it through the root; root, quotient, products."""
    r = x.cpu().double() + (residual.cpu().double() if residual is not None else 0.0)
    if residual is not None:
        r32 = (x.cpu().float() + residual.cpu().float()).double()  # the kernel's sum is one fp32 addition
        r = torch.where(torch.isfinite(r32), r32, r)
    inv = 1.0 / torch.sqrt((r * r).mean(1) + eps)
    return r, inv, r * inv[:, None] * weight.cpu().double(), 40 * U32
