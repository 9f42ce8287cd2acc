"""AdamW over a list of tensors, the step after GradientClipKernel's.

The reference has no counterpart.  As in training.py, ``encode`` takes device tensors, checks them and enqueues on the
context's stream; ``step`` orders the call after torch's current stream and waits.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np

from . import _lib
from .context import GPUContext, VectorError
from .training import _DTYPES, _dtype, _torch, _vector

GROUP = 256  # values of an 8-bit moment that share a scale
_ENTRY = np.dtype([(name, {C.c_void_p: np.uint64, C.c_uint64: np.uint64, C.c_int32: np.int32, C.c_float: np.float32}[kind]) for name, kind in _lib.AdamWTensorDesc._fields_], align=True)


@dataclass
class AdamWState:
    """The moments of a list of tensors, a tensor of each: fp32 m and v, or float8_e4m3fn codes of m and of sqrt(v) with
    fp32 scales [ceil(size / 256)]; and the parameters' 32-bit copies (None: none; None in the list: that one has none)."""

    first: list
    second: list
    firstScales: list | None = None
    secondScales: list | None = None
    masters: list | None = None


class AdamWTensors:
    """Device tensors of a step, listed once: their addresses, sizes and types lie in device memory.  The tensors
    are kept alive; one that is replaced (not written in place) needs a new list."""

    def __init__(self, context: GPUContext, parameters, gradients, state: AdamWState, outputs=None, rateFactors=None, decayFactors=None):
        torch = _torch()
        self._h = None
        self.context, device = context, context.device
        parameters, gradients = list(parameters), list(gradients)
        n = len(parameters)
        wide = state.firstScales is None and state.secondScales is None
        if not wide and (state.firstScales is None or state.secondScales is None):
            raise VectorError.invalidInput("8-bit moments have scales, both of them")
        out_parameters, out_state = outputs if outputs is not None else (parameters, state)
        rates, decays = (list(f) if f is not None else [1.0] * n for f in (rateFactors, decayFactors))
        for name, values in (("gradients", gradients), ("outputs", out_parameters), ("rateFactors", rates), ("decayFactors", decays)):
            if len(values) != n:
                raise VectorError.invalidInput(f"{n} parameters and {len(values)} {name}")
        for name in ("first", "second", "firstScales", "secondScales", "masters"):
            mine, theirs = getattr(state, name), getattr(out_state, name)
            if (mine is None) != (theirs is None):
                raise VectorError.invalidInput(f"{name}: either in the state and the outputs, or in neither")
            for values in (mine, theirs):
                if values is not None and len(values) != n:
                    raise VectorError.invalidInput(f"{n} parameters and {len(values)} {name}")
        kind = torch.float32 if wide else torch.float8_e4m3fn
        for name, tensors in (("parameter", parameters), ("gradient", gradients)):
            for i, t in enumerate(tensors):
                if not torch.is_tensor(t):
                    raise VectorError.invalidInput(f"{name} {i}: expected a tensor, got {type(t).__name__}")
        sizes = [p.numel() for p in parameters]
        groups = [-(-size // GROUP) for size in sizes]

        def pointers(tensors, name, dtypes, counts):
            """Addresses of contiguous tensors of the given types and sizes on the context's device (0 for None)."""
            found = [0] * n
            for i, t in enumerate(tensors):
                if t is None:
                    continue
                if t.dtype == dtypes[i] and t.numel() == counts[i] and t.get_device() == device and t.is_contiguous():
                    found[i] = t.data_ptr()
                else:
                    _vector(t, f"{name} {i}", dtypes[i], counts[i], device)
            return found

        types = [_DTYPES.get(p.dtype) for p in parameters]
        grad_types = [_DTYPES.get(g.dtype) for g in gradients]
        for i, p in enumerate(parameters):
            if types[i] is None or grad_types[i] is None:
                _dtype(p, f"parameter {i}"), _dtype(gradients[i], f"gradient {i}")
            if gradients[i].dtype not in (p.dtype, torch.float32):
                raise VectorError.invalidInput(f"gradient {i}: expected {p.dtype} or float32, got {gradients[i].dtype}")
        table = np.zeros(n, dtype=_ENTRY)
        own, kinds, fp32 = [p.dtype for p in parameters], [kind] * n, [torch.float32] * n
        table["param"], table["out_param"] = pointers(parameters, "parameter", own, sizes), pointers(out_parameters, "output", own, sizes)
        table["grad"] = pointers(gradients, "gradient", [g.dtype for g in gradients], sizes)
        for at, of in (("", state), ("out_", out_state)):
            table[at + "first"], table[at + "second"] = pointers(of.first, "first moment", kinds, sizes), pointers(of.second, "second moment", kinds, sizes)
            if not wide:
                table[at + "first_scales"], table[at + "second_scales"] = pointers(of.firstScales, "scales", fp32, groups), pointers(of.secondScales, "scales", fp32, groups)
            if of.masters is not None:
                table[at + "master"] = pointers(of.masters, "master", fp32, sizes)
        if state.masters is not None and any((a is None) != (b is None) for a, b in zip(state.masters, out_state.masters)):
            raise VectorError.invalidInput("masters: either in the state and the outputs, or in neither")
        table["size"], table["param_dtype"], table["grad_dtype"] = sizes, types, grad_types
        table["rate_factor"], table["decay_factor"] = rates, decays
        keep = [parameters, gradients, list(out_parameters)]
        for s in (state, out_state):
            keep += [list(v) for v in (s.first, s.second, s.firstScales, s.secondScales, s.masters) if v is not None]
        self.tensors = keep
        h = C.c_void_p()
        context.check(context.lib.va_adamw_list_create(context.handle, table.ctypes.data if n else None, n, 32 if wide else 8, C.byref(h)), "va_adamw_list_create")
        self._lib, self._h = context.lib, h

    @property
    def handle(self) -> C.c_void_p:
        if self._h is None:
            raise VectorError("computeFailed", "list destroyed")
        return self._h

    def close(self) -> None:
        """Frees the device's list; waits for the device."""
        if getattr(self, "_h", None) is not None:
            self._lib.va_adamw_list_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class AdamWKernel:
    """One AdamW step of all tensors of a list in one launch.

    With t the step (from 1) and g the gradients, scaled by ``gradScale`` and, where ``gradNorm`` is given (the norm of all
    gradients as GradientClipKernel writes it, before gradScale), clipped to ``maxNorm``:

        m = beta1 m + (1 - beta1) g        v = beta2 v + (1 - beta2) g^2
        p = p (1 - rate weightDecay) - rate m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + epsilon)

    in fp32 throughout, the new parameters rounded once.  With a gradNorm that is not finite nothing changes.
    Parameters are float32, float16 or bfloat16, types may be mixed, gradients of the parameter's type or float32; fp16
    and bf16 parameters may have 32-bit copies (``masters``), without which steps below half of their spacing are
    lost.  Moments are fp32, or 8-bit codes whose rounding is random in proportion (AdamWState): the same
    ``seed``, step and list give the same bits.
    """

    name = "AdamWKernel"

    def __init__(self, context: GPUContext):
        self.context = context

    def state(self, parameters, bits: int = 32, masters: bool = False) -> AdamWState:
        """The state before the first step: moments of zero, and 32-bit copies of the parameters that are not float32."""
        torch = _torch()
        if bits not in (8, 32):
            raise VectorError.invalidInput(f"moments of {bits} bits (8 or 32)")
        parameters = list(parameters)
        zeros = lambda dtype, per=1: [torch.zeros(-(-p.numel() // per), dtype=dtype, device=p.device) for p in parameters]  # noqa: E731
        kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
        copies = [p.detach().float().reshape(-1) if p.dtype != torch.float32 else None for p in parameters] if masters else None
        s = AdamWState(zeros(kind), zeros(kind), masters=copies)
        if bits == 8:
            s.firstScales, s.secondScales = zeros(torch.float32, GROUP), zeros(torch.float32, GROUP)
        return s

    def tensorList(self, parameters, gradients, state: AdamWState, outputs=None, rateFactors=None, decayFactors=None) -> AdamWTensors:
        """The list of a step, in place or into ``outputs`` (parameters and an AdamWState); rateFactors and decayFactors: a
        factor of each tensor's rate and weight decay.  Allocates and waits; refused while the context's stream is captured."""
        return AdamWTensors(self.context, parameters, gradients, state, outputs, rateFactors, decayFactors)

    def encode(self, tensors: AdamWTensors, step, learningRate, beta1: float = 0.9, beta2: float = 0.999, epsilon: float = 1e-8,
               weightDecay: float = 0.01, gradNorm=None, maxNorm: float | None = None, gradScale: float = 1.0, seed: int = 0) -> None:
        """step: a number, or one int64 value on the device; learningRate: a number, or one float32 value on the device (a
        captured step reads both anew)."""
        c, torch = self.context, _torch()
        if tensors.context.device != c.device:
            raise VectorError.invalidInput(f"tensors: on cuda:{tensors.context.device}, expected cuda:{c.device}")
        if maxNorm is not None and gradNorm is None:
            raise VectorError.invalidInput("clipping needs the gradients' norm")
        p = _lib.AdamWParams()
        if isinstance(step, torch.Tensor):
            p.device_step = _vector(step, "step", torch.int64, 1, c.device)
        else:
            p.step = int(step)
        if isinstance(learningRate, torch.Tensor):
            p.device_rate = _vector(learningRate, "learningRate", torch.float32, 1, c.device)
        else:
            p.rate = float(learningRate)
        if gradNorm is not None:
            p.grad_norm = _vector(gradNorm, "gradNorm", torch.float32, 1, c.device)
        p.max_norm = float(maxNorm) if maxNorm is not None else float("inf")
        p.beta1, p.beta2, p.epsilon, p.weight_decay, p.grad_scale = float(beta1), float(beta2), float(epsilon), float(weightDecay), float(gradScale)
        p.seed = int(seed) & 0xFFFFFFFFFFFFFFFF
        c.check(c.lib.va_adamw_step(c.handle, tensors.handle, C.byref(p)), "va_adamw_step")

    def step(self, tensors: AdamWTensors, step, learningRate, **settings) -> None:
        """encode, after torch's current stream; waits."""
        c = self.context
        c.order_after_torch()
        self.encode(tensors, step, learningRate, **settings)
        c.synchronize()
