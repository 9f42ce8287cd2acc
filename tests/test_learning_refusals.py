"""Refusals of the optimizer, of the microscaled rows and of sampling that need no device: a NULL context at the C
boundary, and what the Python classes check before they call.  No kernel is launched here."""
from __future__ import annotations

import ctypes as C
import subprocess

import pytest
import torch

from vectoraccelerate_amd import AdamWKernel, AdamWState, MicroscaledQuantizationKernel, MicroscaledRows, SoftmaxSamplingKernel, VectorError, _lib


class NoDevice:
    """A context for calls that have to end before they reach it."""

    device = 0

    def __getattr__(self, name):
        raise AssertionError(f"the call went on to the context ({name})")


@pytest.fixture(scope="module")
def lib():
    from vectoraccelerate_amd import build as b

    if not _lib.LIB_PATH.exists():
        b.build()
    return _lib.load()


def test_null_context(lib):
    t, p, r, s = _lib.AdamWTensorDesc(), _lib.AdamWParams(), _lib.MxRowsDesc(), _lib.SampleDesc()
    h = C.c_void_p()
    assert lib.va_adamw_list_create(None, C.addressof(t), 1, 32, C.byref(h)) == 1 and not h
    assert lib.va_adamw_list_destroy(None) == 1
    assert lib.va_adamw_step(None, None, C.byref(p)) == 1
    assert lib.va_mx_quantize(None, None, 1, 0, C.byref(r)) == 1
    assert lib.va_mx_dequantize(None, C.byref(r), 0, None, 1) == 1
    assert lib.va_mx_product(None, C.byref(r), C.byref(r), 1.0, None, 0, None, 1) == 1
    assert lib.va_mx_product_rows(None, None, 1, 0, 1, C.byref(r), 1.0, None, 0, None, 1) == 1
    assert lib.va_sample(None, C.byref(s), None, None) == 1
    assert lib.va_sample_workspace(None, 4, 100_000) == 0


def test_descriptions_match_the_header():
    """Sizes of the C structs on a 64-bit host."""
    assert C.sizeof(_lib.AdamWTensorDesc) == 13 * 8 + 8 + 4 * 4
    assert C.sizeof(_lib.AdamWParams) == 3 * 8 + 2 * 8 + 7 * 8
    assert C.sizeof(_lib.MxRowsDesc) == 4 * 8 + 2 * 4
    assert C.sizeof(_lib.SampleDesc) == 6 * 8 + 8 + 7 * 4 + 4 + 2 * 8


def _state(p, bits=32, masters=None):
    kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
    z = lambda: [torch.zeros(t.numel()).to(kind) for t in p]  # noqa: E731
    s = lambda: [torch.zeros(-(-t.numel() // 256)) for t in p] if bits == 8 else None  # noqa: E731
    return AdamWState(z(), z(), s(), s(), masters)


def test_host_tensors_are_refused():
    c = NoDevice()
    x, out, n = torch.zeros(4, 8), torch.zeros(4, 4), torch.zeros(4)
    rows = MicroscaledRows(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 8)
    micro, sampling = MicroscaledQuantizationKernel(c), SoftmaxSamplingKernel(c)
    items = torch.zeros(4, dtype=torch.int64)
    for f in (lambda: AdamWKernel(c).tensorList([x], [x], _state([x])), lambda: AdamWKernel(c).tensorList([x], [x], _state([x], 8)),
              lambda: micro.encodeQuantize(x, rows), lambda: micro.encodeDequantize(rows, x), lambda: micro.encodeProduct(rows, rows, out),
              lambda: micro.encodeProduct(x, rows, out), lambda: sampling.encode(x, n, items), lambda: sampling.encode(x.double(), n, items)):
        with pytest.raises(VectorError):
            f()


def test_lists_are_checked():
    k, p = AdamWKernel(NoDevice()), [torch.zeros(8), torch.zeros(3)]
    s = _state(p)
    eight = _state(p, 8)
    for f in (lambda: k.tensorList(p, p[:1], s), lambda: k.tensorList(p, [p[0], None], s), lambda: k.tensorList([p[0], None], p, s),
              lambda: k.tensorList(p, p, AdamWState(s.first, s.second[:1])), lambda: k.tensorList(p, p, AdamWState(eight.first, eight.second, eight.firstScales)),
              lambda: k.tensorList(p, p, s, outputs=(p, _state(p, masters=[None, None]))), lambda: k.tensorList(p, p, s, outputs=(p[:1], s)),
              lambda: k.tensorList(p, p, s, rateFactors=[1.0]), lambda: k.tensorList(p, p, s, decayFactors=[1.0] * 3),
              lambda: k.state(p, 16), lambda: k.tensorList([t.double() for t in p], p, s)):
        with pytest.raises(VectorError):
            f()


def test_dimensions_and_counts_are_checked():
    micro, sampling = MicroscaledQuantizationKernel(NoDevice()), SoftmaxSamplingKernel(NoDevice())
    codes = torch.zeros(4, 64, dtype=torch.uint8)
    for f in (lambda: micro.encodeQuantize(torch.zeros(4, 0), MicroscaledRows(codes, codes[:, :4], 0)),
              lambda: micro.encodeQuantize(torch.zeros(4, 200), MicroscaledRows(codes, codes[:, :4], 200)),
              lambda: sampling.encode(torch.zeros(4), torch.zeros(4), torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(VectorError):
            f()


def test_a_list_is_not_made_while_its_stream_is_captured(lib, tmp_path):
    """tests/cpp/capture_host.cpp, whose runtime is host memory: a refusal before anything is allocated or copied."""
    root = _lib.LIB_PATH.parent.parent
    exe = tmp_path / "capture_host"
    cmd = ["g++", "-std=c++17", "-O1", "-rdynamic", f"-I{root / 'include'}", "-I/opt/rocm/include", str(root / "tests" / "cpp" / "capture_host.cpp"), f"-L{_lib.LIB_PATH.parent}",
           "-lva_hip", f"-Wl,-rpath,{_lib.LIB_PATH.parent}", "-Wl,-rpath-link,/opt/rocm/lib", "-o", str(exe)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "ok" in run.stdout, run.stdout + run.stderr


def test_an_order_needs_a_context(lib):
    for order in (0, 1, 2):
        assert lib.va_sample_in_order(None, C.byref(_lib.SampleDesc()), order, None, None) == 1
    sampling = SoftmaxSamplingKernel(NoDevice())
    for order in ("", "falling", None):
        with pytest.raises(VectorError):
            sampling.encode(torch.zeros(4, 4), torch.zeros(4), torch.zeros(4, dtype=torch.int64), order=order)
