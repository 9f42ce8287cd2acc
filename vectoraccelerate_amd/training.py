"""Training and serving of the embeddings that a collection holds.

SoftmaxCrossEntropyKernel  the loss of hidden rows against every item of a collection, and its gradient
RMSNormKernel              root-mean-square norm with the residual's addition, its backward pass, and
                           its output in 8 bits with scales (the codes of the int8 scan)
GradientClipKernel         the global norm of a list of gradients, and the gradients clipped by it

The reference has no counterpart of these.  They follow its kernel classes: ``encode*`` takes device
tensors, checks them and enqueues on the context's stream (inputs must be ready for that stream, and
tensors must live until the work is done); the other methods allocate the outputs, order the call after
torch's current stream and wait.  All arithmetic runs in libva_hip.so.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

from . import _lib
from .context import GPUContext, VectorError, dptr

_REDUCTIONS = {"mean": _lib.VA_REDUCE_MEAN, "sum": _lib.VA_REDUCE_SUM, "none": _lib.VA_REDUCE_NONE}
_DTYPES: dict = {}
_CODES: dict = {}


def _torch():
    import torch

    if not _DTYPES:
        _DTYPES.update({torch.float32: _lib.VA_DTYPE_F32, torch.float16: _lib.VA_DTYPE_F16, torch.bfloat16: _lib.VA_DTYPE_BF16})
        _CODES.update({torch.int8: _lib.VA_CODE_INT8, torch.float8_e4m3fn: _lib.VA_CODE_FP8_E4M3})
    return torch


def _dtype(t, name: str) -> int:
    _torch()
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise VectorError.invalidInput(f"{name}: unsupported type {t.dtype} (float32, float16 or bfloat16)")
    return d


def _place(t, name: str, device: int) -> None:
    got = t.get_device()  # -1 on the CPU
    if got != device:
        raise VectorError.invalidInput(f"{name}: expected a device (CUDA) tensor" if got < 0 else f"{name}: on {t.device}, expected cuda:{device}")


def _rows(t, name: str, device: int, dtype=None, shape=None) -> tuple[int, int]:
    """(device pointer, elements between rows) of a matrix on the context's device whose rows are
    contiguous; checked against `dtype` and `shape`."""
    _place(t, name, device)
    got = t.shape
    if len(got) != 2:
        raise VectorError.invalidInput(f"{name}: expected a matrix, got {len(got)} dimensions")
    rows, dim = got
    if shape is not None and got != shape:
        if dim != shape[1]:
            raise VectorError.dimensionMismatch(shape[1], dim)
        raise VectorError.invalidInput(f"{name}: expected {shape[0]} rows, got {rows}")
    if dtype is not None and t.dtype != dtype:
        raise VectorError.invalidInput(f"{name}: expected {dtype}, got {t.dtype}")
    sr, sd = t.stride()
    if sd != 1 and dim > 1:
        raise VectorError.invalidInput(f"{name}: the values of a row must be contiguous")
    if rows < 2:
        return t.data_ptr(), dim  # (one row has no stride, whatever the tensor's view says)
    if sr < dim:
        raise VectorError.invalidInput(f"{name}: rows overlap")
    return t.data_ptr(), sr


def _vector(t, name: str, dtype, count: int, device: int) -> int:
    """Device pointer of a contiguous vector of `count` values of `dtype` on the context's device."""
    if t.dtype != dtype or t.numel() != count or t.get_device() != device or not t.is_contiguous():
        raise VectorError.invalidInput(
            f"{name}: expected {count} contiguous values of {dtype} on cuda:{device}, got {tuple(t.shape)} of {t.dtype} on {t.device}")
    return t.data_ptr()


@dataclass
class SoftmaxCrossEntropyResult:
    """Device tensors: per-row loss and log-sum-exp, and the reduced loss (None without a reduction)."""

    loss: object
    logSumExp: object
    reduced: object


class SoftmaxCrossEntropyKernel:
    """Softmax cross entropy of hidden rows [T x D] over all items [V x D] of a collection.

    logits = scale * hidden @ items.T + offsets;  loss_t = logsumexp(logits_t) - logits_t[target_t].
    The logits are never stored.  offsets (fp32 [V] or None) are constants: corrections of a sampled
    softmax, and -inf for deleted items, which have no probability and no gradient whatever their
    vectors hold.  Rows whose target is ``ignoreIndex`` have loss 0 and gradient 0; a target outside
    the collection gives a NaN loss and gradient 0.  Targets are int64.  hidden and items are float32,
    float16 or bfloat16 alike, their rows may be strided.

    Sums are fp32.  In 16 bits the logits' gradients are rounded once to the type before they are summed
    into the results.  In float32 more than 32 rows (64 over 65,536 items and more) enter the logits
    as two float16 values each: exact to 2^-22 of the value or 2^-39 of the largest of its row.
    """

    name = "SoftmaxCrossEntropyKernel"

    def __init__(self, context: GPUContext):
        self.context = context

    def _describe(self, hidden, items, targets, scale, offsets, ignoreIndex):
        torch, device = _torch(), self.context.device
        dtype = _dtype(hidden, "hidden")
        hp, hs = _rows(hidden, "hidden", device)
        T, D = hidden.shape
        ip, is_ = _rows(items, "items", device, hidden.dtype)
        V, width = items.shape
        if width != D:
            raise VectorError.dimensionMismatch(D, width)
        return _lib.XentDesc(hp, ip, _vector(targets, "targets", torch.int64, T, device),
                             _vector(offsets, "offsets", torch.float32, V, device) if offsets is not None else None,
                             hs, is_, int(ignoreIndex), T, V, D, dtype, float(scale))

    def encodeForward(self, hidden, items, targets, outLoss, outLogSumExp, outReduced=None, reduction: str = "mean",
                      scale: float = 1.0, offsets=None, ignoreIndex: int = -100) -> None:
        """outLoss and outLogSumExp: fp32 [T]; outReduced (one fp32 value or None): the reduced loss."""
        c, f32 = self.context, _torch().float32
        d = self._describe(hidden, items, targets, scale, offsets, ignoreIndex)
        mode = _reduction(reduction) if outReduced is not None else _lib.VA_REDUCE_NONE
        if outReduced is not None and mode == _lib.VA_REDUCE_NONE:
            raise VectorError.invalidInput("a reduced loss needs a reduction")
        c.check(c.lib.va_xent_forward(c.handle, C.byref(d), _vector(outLoss, "outLoss", f32, d.rows, c.device),
                                      _vector(outLogSumExp, "outLogSumExp", f32, d.rows, c.device), mode,
                                      _vector(outReduced, "outReduced", f32, 1, c.device) if outReduced is not None else None),
                "va_xent_forward")

    def encodeBackward(self, hidden, items, targets, logSumExp, outGradHidden=None, outGradItems=None, grad=None,
                       reduction: str = "mean", scale: float = 1.0, offsets=None, ignoreIndex: int = -100) -> None:
        """Gradients of the reduced loss times ``grad`` (one fp32 value; None: 1), or with reduction "none"
        of sum(grad * loss) for grad of [T].  logSumExp is encodeForward's; the outputs have the
        type and shape of what they are the gradient of, and either may be None."""
        c, f32 = self.context, _torch().float32
        d = self._describe(hidden, items, targets, scale, offsets, ignoreIndex)
        mode = _reduction(reduction)
        if mode == _lib.VA_REDUCE_NONE and grad is None:
            raise VectorError.invalidInput("without a reduction the rows' gradients are needed")
        count = d.rows if mode == _lib.VA_REDUCE_NONE else 1
        hp, hs = _rows(outGradHidden, "outGradHidden", c.device, hidden.dtype, hidden.shape) if outGradHidden is not None else (None, 0)
        ip, is_ = _rows(outGradItems, "outGradItems", c.device, hidden.dtype, items.shape) if outGradItems is not None else (None, 0)
        c.check(c.lib.va_xent_backward(c.handle, C.byref(d), _vector(logSumExp, "logSumExp", f32, d.rows, c.device), mode,
                                       _vector(grad, "grad", f32, count, c.device) if grad is not None else None, hp, hs, ip, is_),
                "va_xent_backward")

    def forward(self, hidden, items, targets, reduction: str = "mean", scale: float = 1.0, offsets=None,
                ignoreIndex: int = -100) -> SoftmaxCrossEntropyResult:
        c, torch = self.context, _torch()
        T, mode = hidden.shape[0], _reduction(reduction)
        loss, lse = c.empty((T,), torch.float32), c.empty((T,), torch.float32)
        reduced = c.empty((1,), torch.float32) if mode != _lib.VA_REDUCE_NONE else None
        c.order_after_torch()
        self.encodeForward(hidden, items, targets, loss, lse, reduced, reduction, scale, offsets, ignoreIndex)
        c.synchronize()
        return SoftmaxCrossEntropyResult(loss, lse, reduced)

    def backward(self, hidden, items, targets, logSumExp, grad=None, reduction: str = "mean", scale: float = 1.0, offsets=None,
                 ignoreIndex: int = -100):
        """(gradient of hidden, gradient of items)."""
        c = self.context
        gh, gi = c.empty(hidden.shape, hidden.dtype), c.empty(items.shape, items.dtype)
        c.order_after_torch()
        self.encodeBackward(hidden, items, targets, logSumExp, gh, gi, grad, reduction, scale, offsets, ignoreIndex)
        c.synchronize()
        return gh, gi


def _reduction(name: str) -> int:
    if name not in _REDUCTIONS:
        raise VectorError.invalidInput(f"unknown reduction {name!r} (mean, sum or none)")
    return _REDUCTIONS[name]


class RMSNormKernel:
    """y = r / sqrt(mean(r^2) + epsilon) * weight with r = x + residual, over rows [T x D].

    x, residual, weight and the outputs are float32, float16 or bfloat16 alike; rows may be strided,
    and an output may be the input that it replaces.  The 8-bit forms write codes (int8, or
    float8_e4m3fn) with a scale for each row (groupSize 0) or for each group of ``groupSize``
    dimensions (a power of two from 8 to 512), or on the one grid of ``givenScale``.
    """

    name = "RMSNormKernel"

    def __init__(self, context: GPUContext):
        self.context = context

    def _describe(self, x, weight, residual, outResidual, outInverseRms, epsilon):
        torch, device = _torch(), self.context.device
        dtype = _dtype(x, "x")
        xp, xs = _rows(x, "x", device)
        T, D = shape = x.shape
        rp, rs = _rows(residual, "residual", device, x.dtype, shape) if residual is not None else (None, 0)
        op, os_ = _rows(outResidual, "outResidual", device, x.dtype, shape) if outResidual is not None else (None, 0)
        ip = _vector(outInverseRms, "outInverseRms", torch.float32, T, device) if outInverseRms is not None else None
        if weight.numel() != D:
            raise VectorError.dimensionMismatch(D, weight.numel())
        return _lib.RmsDesc(xp, rp, _vector(weight, "weight", x.dtype, D, device), op, ip, xs, rs, os_, T, D, dtype, float(epsilon))

    def _codes(self, codes, shape):
        _torch()
        code = _CODES.get(codes.dtype)
        if code is None:
            raise VectorError.invalidInput(f"codes: unsupported type {codes.dtype} (int8 or float8_e4m3fn)")
        p, s = _rows(codes, "codes", self.context.device, None, shape)
        return code, p, s

    def _scales(self, scales, givenScale, groupSize, T, D):
        if (scales is None) == (givenScale is None):
            raise VectorError.invalidInput("either scales or a given scale")
        if givenScale is not None:
            if not float(givenScale) > 0.0:
                raise VectorError.invalidInput(f"a given scale must be positive, got {givenScale}")
            return None
        groups = -(-D // groupSize) if groupSize else 1
        return _vector(scales, "scales", _torch().float32, T * groups, self.context.device)

    def encode(self, x, weight, out, residual=None, outResidual=None, outInverseRms=None, epsilon: float = 1e-6) -> None:
        c = self.context
        d = self._describe(x, weight, residual, outResidual, outInverseRms, epsilon)
        op, os_ = _rows(out, "out", c.device, x.dtype, x.shape)
        c.check(c.lib.va_rms_norm(c.handle, C.byref(d), op, os_), "va_rms_norm")

    def encodeQuantized(self, x, weight, outCodes, outScales=None, residual=None, outResidual=None, outInverseRms=None,
                        groupSize: int = 0, givenScale: float | None = None, epsilon: float = 1e-6) -> None:
        c = self.context
        d = self._describe(x, weight, residual, outResidual, outInverseRms, epsilon)
        code, cp, cs = self._codes(outCodes, x.shape)
        sp = self._scales(outScales, givenScale, groupSize, d.rows, d.dim)
        c.check(c.lib.va_rms_norm_quantized(c.handle, C.byref(d), code, int(groupSize), float(givenScale or 0.0), cp, cs, sp),
                "va_rms_norm_quantized")

    def encodeDequantize(self, codes, scales, out, groupSize: int = 0, givenScale: float | None = None) -> None:
        """out = code * scale in out's type."""
        c = self.context
        dtype = _dtype(out, "out")
        op, os_ = _rows(out, "out", c.device)
        T, D = out.shape
        code, cp, cs = self._codes(codes, out.shape)
        sp = self._scales(scales, givenScale, groupSize, T, D)
        c.check(c.lib.va_rms_dequantize(c.handle, cp, cs, code, sp, float(givenScale or 0.0), T, D, int(groupSize), dtype, op, os_),
                "va_rms_dequantize")

    def encodeBackward(self, grad, summed, weight, inverseRms, outGradX=None, outGradWeight=None, gradResidual=None) -> None:
        """``summed`` is x + residual as the forward pass stored it (x where there was no residual), inverseRms
        its outInverseRms, gradResidual what reaches the new residual from behind.  outGradX is the
        gradient of x and of the residual alike."""
        c = self.context
        d = self._describe(summed, weight, None, None, None, 0.0)
        dtype, shape = summed.dtype, summed.shape
        gp, gs = _rows(grad, "grad", c.device, dtype, shape)
        rp, rs = _rows(gradResidual, "gradResidual", c.device, dtype, shape) if gradResidual is not None else (None, 0)
        xp, xs = _rows(outGradX, "outGradX", c.device, dtype, shape) if outGradX is not None else (None, 0)
        wp = _vector(outGradWeight, "outGradWeight", dtype, d.dim, c.device) if outGradWeight is not None else None
        c.check(c.lib.va_rms_norm_backward(c.handle, C.byref(d), gp, gs, rp, rs,
                                           _vector(inverseRms, "inverseRms", _torch().float32, d.rows, c.device), xp, xs, wp),
                "va_rms_norm_backward")

    def forward(self, x, weight, residual=None, epsilon: float = 1e-6):
        """(y, x + residual, inverse rms)."""
        c, torch = self.context, _torch()
        y, r = c.empty(x.shape, x.dtype), c.empty(x.shape, x.dtype) if residual is not None else x
        inv = c.empty((x.shape[0],), torch.float32)
        c.order_after_torch()
        self.encode(x, weight, y, residual, r if residual is not None else None, inv, epsilon)
        c.synchronize()
        return y, r, inv

    def quantize(self, x, weight, residual=None, code=None, groupSize: int = 0, givenScale: float | None = None, epsilon: float = 1e-6):
        """(codes, scales or None, x + residual); code: torch.int8 (the default) or torch.float8_e4m3fn."""
        c, torch = self.context, _torch()
        T, D = x.shape
        codes = c.empty((T, D), code or torch.int8)
        scales = c.empty((T, -(-D // groupSize) if groupSize else 1), torch.float32) if givenScale is None else None
        r = c.empty(x.shape, x.dtype) if residual is not None else x
        c.order_after_torch()
        self.encodeQuantized(x, weight, codes, scales, residual, r if residual is not None else None, None, groupSize, givenScale, epsilon)
        c.synchronize()
        return codes, scales, r

    def backward(self, grad, summed, weight, inverseRms, gradResidual=None):
        """(gradient of x and of the residual, gradient of weight)."""
        c = self.context
        gx, gw = c.empty(summed.shape, summed.dtype), c.empty(weight.shape, weight.dtype)
        c.order_after_torch()
        self.encodeBackward(grad, summed, weight, inverseRms, gx, gw, gradResidual)
        c.synchronize()
        return gx, gw


class TensorList:
    """Device tensors of a call, listed once: their addresses, sizes and types.  The tensors are kept
    alive; a tensor that is replaced (not written in place) needs a new list."""

    def __init__(self, tensors, outputs=None):
        _torch()
        self.tensors = list(tensors)
        self.outputs = list(outputs) if outputs is not None else None
        if self.outputs is not None and len(self.outputs) != len(self.tensors):
            raise VectorError.invalidInput(f"{len(self.tensors)} tensors and {len(self.outputs)} outputs")
        for i, t in enumerate(self.tensors):
            _dtype(t, f"tensor {i}")
            dptr(t)
            if t.device != self.tensors[0].device:
                raise VectorError.invalidInput(f"tensor {i}: on {t.device}, expected {self.tensors[0].device}")
            if self.outputs is not None:
                o = self.outputs[i]
                dptr(o)
                if o.dtype != t.dtype or o.numel() != t.numel() or o.device != t.device:
                    raise VectorError.invalidInput(f"output {i}: expected {t.numel()} values of {t.dtype} on {t.device}")
        n = len(self.tensors)
        self._in = (C.c_void_p * n)(*[t.data_ptr() for t in self.tensors])
        self._out = (C.c_void_p * n)(*[t.data_ptr() for t in self.outputs]) if self.outputs is not None else None
        self._sizes = (C.c_uint64 * n)(*[t.numel() for t in self.tensors])
        self._dtypes = (C.c_int32 * n)(*[_DTYPES[t.dtype] for t in self.tensors])
        cast = lambda a: C.cast(a, C.c_void_p) if a is not None else None  # noqa: E731
        self.desc = _lib.TensorListDesc(cast(self._in), cast(self._out), cast(self._sizes), cast(self._dtypes), n)


class GradientClipKernel:
    """norm = sqrt(sum of the squares of all values of a list of tensors); every tensor times
    min(1, maxNorm / (norm + epsilon)), in place or into the list's outputs.  Types may be mixed; a tensor is
    listed once."""

    name = "GradientClipKernel"

    def __init__(self, context: GPUContext):
        self.context = context

    def tensorList(self, tensors, outputs=None) -> TensorList:
        return TensorList(tensors, outputs)

    def encode(self, tensors: TensorList, maxNorm: float, outNorm=None, epsilon: float = 1e-6) -> None:
        """outNorm: one fp32 value on the device, or None."""
        c = self.context
        if tensors.tensors:
            _place(tensors.tensors[0], "tensors", c.device)  # (the list has checked that they are together)
        norm = _vector(outNorm, "outNorm", _torch().float32, 1, c.device) if outNorm is not None else None
        c.check(c.lib.va_grad_clip(c.handle, C.byref(tensors.desc), float(maxNorm), float(epsilon), norm), "va_grad_clip")

    def clip(self, tensors, maxNorm: float, epsilon: float = 1e-6) -> float:
        """Clips the tensors in place and returns their norm before."""
        c = self.context
        norm = c.empty((1,), _torch().float32)
        c.order_after_torch()
        self.encode(TensorList(tensors), maxNorm, norm, epsilon)
        c.synchronize()
        return float(norm.item())
