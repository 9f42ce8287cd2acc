"""The training and serving operators together: the example that trains a collection's embeddings, codes and
searches them, and the C++ classes (run by tests/cpp/va_example) against the definitions in 64 bits."""
from __future__ import annotations

import importlib.util
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from tests import training_oracle as oracle
from tests.training_oracle import U32

ROOT = Path(__file__).resolve().parent.parent
EXE = ROOT / "tests" / "cpp" / "va_example"
pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("train_and_serve", ROOT / "examples" / "train_and_serve.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_train_and_serve(ctx, dtype):
    """Training halves the loss of a uniform guess and the int8 search finds the queries' items."""
    items = 2000
    r = _example().run(ctx, items=items, dim=64, batch=512, steps=40, dtype=dtype)
    assert np.isfinite(r["losses"]).all() and np.isfinite(r["norms"]).all()
    assert abs(r["losses"][0] - np.log(items)) < 0.5  # small random logits over the items
    assert r["losses"][-1] < 0.5 * r["losses"][0]
    assert r["target_in_top10"] > 0.8 and r["top10_agreement"] > 0.8


def test_cpp_classes(tmp_path):
    if not EXE.exists():
        from vectoraccelerate_amd.build import build_cpp_example

        build_cpp_example()
    Q, N, D, C = 40, 1500, 32, 8
    g = np.random.default_rng(3)
    q, x, c = (g.standard_normal((n, D), np.float32) for n in (Q, N, C))
    for name, arr in (("q", q), ("x", x), ("c", c)):
        arr.tofile(tmp_path / f"{name}.bin")
    proc = subprocess.run([str(EXE), str(tmp_path), str(Q), str(N), str(D), str(C), "5", "4"], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stderr
    rd = lambda n, shape: torch.from_numpy(np.fromfile(tmp_path / f"{n}.bin", np.float32)).view(*shape)  # noqa: E731
    tq, tx = torch.from_numpy(q), torch.from_numpy(x)
    want = oracle.xent(tq, tx, torch.arange(Q), 0.25, None, -100, torch.full((Q,), 1.0 / Q, dtype=torch.float64))
    oracle.close(rd("xent_loss", (Q,)), *want["loss"], "loss")
    loss, bound = want["loss"]
    oracle.close(rd("xent_mean", (1,)), loss.mean().view(1), (bound.mean() + 2 * U32 * loss.abs().mean()).view(1), "mean")
    (gq, eq), (gx, ex) = want["grad_hidden"], want["grad_items"]
    norm = torch.sqrt((gq * gq).sum() + (gx * gx).sum())
    off = torch.sqrt((eq * eq).sum() + (ex * ex).sum())  # the norm moves by at most its gradients' errors' norm
    oracle.close(rd("clip_norm", (1,)), norm.view(1), (off + 2 * U32 * norm).view(1), "norm")
    f = min(1.0, 0.01 / (float(norm) + 1e-6))
    assert f < 1.0
    slack = float(off / norm) + 4 * U32
    oracle.close(rd("clip_gq", (Q, D)), gq * f, (eq + gq.abs() * slack) * f, "clipped")
    oracle.close(rd("clip_gx", (N, D)), gx * f, (ex + gx.abs() * slack) * f, "clipped")
    w = torch.full((D,), 0.5)
    _, inv, y, e = oracle.rms(tq, None, w, 1e-6)
    oracle.close(rd("rms_y", (Q, D)), y, (e + U32) * y.abs(), "y")
    step = y.abs().amax(1, keepdim=True) / 127.0
    oracle.close(rd("rms_back", (Q, D)), y, step * (0.5 + 127.0 * (2 * e + 8 * U32)), "codes")
    n = tq.double() * inv[:, None]
    gy = 0.5 * y
    gr = inv[:, None] * (gy - n * (gy * n).mean(1, keepdim=True))
    # (y as the gradient is off by e of itself; the row's mean by as much of its magnitudes)
    oracle.close(rd("rms_gr", (Q, D)), gr, inv[:, None] * (gy.abs() + n.abs() * (gy * n).abs().mean(1, keepdim=True)) * (4 * e), "gradient")
