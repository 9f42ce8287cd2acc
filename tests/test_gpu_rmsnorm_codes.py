"""The 8-bit codes of the RMS norm are the roundings of the fp32 quotients y / s, midpoints included."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _midpoints(code, count, generator):
    """Values halfway between two neighbouring codes, and their fp32 neighbours; below the largest code."""
    if code == torch.int8:
        k = torch.randint(0, 126, (count,), generator=generator).float() + 0.5
    else:
        # e4m3 codes between 2^-6 and 416 are 8 to a power of two
        e = torch.randint(-6, 8, (count,), generator=generator)
        k = (8.5 + torch.randint(0, 8, (count,), generator=generator)) * 2.0 ** (e - 3)
    up = torch.randint(-1, 2, (count,), generator=generator)
    k = torch.where(up == 0, k, torch.nextafter(k, torch.where(up > 0, torch.tensor(1e9), torch.tensor(0.0))))
    return k * torch.where(torch.rand(count, generator=generator) < 0.5, -1.0, 1.0)


def _expected(y, s, code):
    """round(y / s) with the quotient an fp32 value, ties to even, saturating."""
    z = torch.from_numpy(y.numpy() / s.numpy())
    if code == torch.int8:
        return torch.from_numpy(np.clip(np.rint(z.numpy()), -127, 127)).to(torch.int8)
    return z.clamp(-448, 448).to(torch.float8_e4m3fn)


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("D", [64, 2048, 4096, 8200])
@pytest.mark.parametrize("form", ["given", "row", "group"])
def test_midpoints(ctx, form, D, code):
    """Rows of +-1 and epsilon 0 have the inverse rms 1, so y is the weight with its sign, exactly: fp32 weights around
    the midpoints of a hundred scales."""
    from vectoraccelerate_amd import RMSNormKernel

    k = RMSNormKernel(ctx)
    g = torch.Generator().manual_seed(D)
    most = 127.0 if code == torch.int8 else 448.0
    x = torch.where(torch.rand(4, D, generator=g) < 0.5, -1.0, 1.0)
    for _ in range(100):
        top = torch.exp(torch.randn((), generator=g) * 8).float()
        s = torch.from_numpy(np.array(top.numpy() / np.float32(most)))
        w = _midpoints(code, D, g) * s
        group = 32 if form == "group" else 0
        w[:: group or D] = top  # the largest magnitude of each group: its scale is s
        codes, scales, _ = k.quantize(x.cuda(), w.cuda(), None, code, group, float(s) if form == "given" else None, 0.0)
        if form != "given":
            assert (scales.cpu() == s).all()
        want = _expected(x * w, s, code)
        assert torch.equal(codes.cpu().view(torch.int8), want.view(torch.int8))
