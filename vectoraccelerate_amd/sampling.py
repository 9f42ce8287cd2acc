"""Items drawn from the softmax over a collection: answers in service, negatives in training.

The reference has no counterpart.  As in training.py, ``encode`` takes device tensors, checks them and enqueues on the
context's stream; ``sample`` allocates the outputs, orders the call after torch's current stream and waits.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .context import GPUContext, VectorError
from .training import _dtype, _rows, _torch, _vector


class SoftmaxSamplingKernel:
    """One item of each row of logits [T x V], float32, float16 or bfloat16, whose rows may be strided.

    With M a row's largest logit, item j weighs exp((x_j - M) / temperature).  Ordered by (logit descending, index ascending)
    topK keeps the first k items (0: all), topP the fewest whose weights add up to p of those that topK keeps, minP
    those that weigh at least minP.  The drawn item is the first, in the order of the items, at which the kept weights added up
    exceed u times their sum; u in [0, 1) is given.  With order "logits" it is the first in the order of the truncations: a smaller u draws
    a more likely item, wherever it lies.  A temperature of 0 draws the most likely item, the first of those as
    likely.  NaN and -inf (a masked item) are never drawn; a row without an item gives -1 and a log probability of -inf.
    Weights and sums are fp64 (a weight is good to 4e-14 of itself; one below 2^-1000 of the largest may count as zero, and an item without
    weight is not drawn); the same inputs give the same items.

    Each setting is one number, or a device tensor with a value for each row (float32, topK int32), where what lies outside a setting's
    range is taken as its nearest value, and NaN as "not truncated" (a temperature: as 0).
    """

    name = "SoftmaxSamplingKernel"
    orders = {"items": 0, "logits": 1}

    def __init__(self, context: GPUContext):
        self.context = context

    def workspaceBytes(self, rows: int, items: int) -> int:
        """Bytes of a workspace for logits of that shape (0: none is used)."""
        return int(self.context.lib.va_sample_workspace(self.context.handle, rows, items))

    def encode(self, logits, uniforms, outItems, outLogProbability=None, temperature=1.0, topK=0, topP=1.0, minP=0.0, workspace=None, order: str = "items") -> None:
        """uniforms: float32 [T]; outItems: int64 [T]; outLogProbability (float32 [T] or None): of the drawn item among those
        that were kept.  workspace (uint8, or None): memory of the call's own in place of the context's scratch arena; a call that is
        captured into a graph without one takes a slower way, and no other call may use it meanwhile."""
        c, torch = self.context, _torch()
        if order not in self.orders:
            raise VectorError.invalidInput(f"order: {order!r} (one of {', '.join(self.orders)})")
        dtype = _dtype(logits, "logits")
        p, stride = _rows(logits, "logits", c.device)
        T, V = logits.shape
        d = _lib.SampleDesc(logits=p, uniforms=_vector(uniforms, "uniforms", torch.float32, T, c.device), stride=stride, rows=T, num_items=V, dtype=dtype,
                            temperature=1.0, top_p=1.0)
        for name, value, one, many, of in (("temperature", temperature, "temperature", "temperatures", torch.float32), ("topK", topK, "top_k", "top_ks", torch.int32),
                                           ("topP", topP, "top_p", "top_ps", torch.float32), ("minP", minP, "min_p", "min_ps", torch.float32)):
            if isinstance(value, torch.Tensor):
                setattr(d, many, _vector(value, name, of, T, c.device))
            elif of == torch.int32:
                if not 0 <= int(value) < 1 << 31:
                    raise VectorError.invalidInput(f"{name}: {value}")
                setattr(d, one, int(value))
            else:
                setattr(d, one, float(value))
        if workspace is not None:
            d.workspace, d.workspace_bytes = _vector(workspace, "workspace", torch.uint8, workspace.numel(), c.device), workspace.numel()
        c.check(c.lib.va_sample_in_order(c.handle, C.byref(d), self.orders[order], _vector(outItems, "outItems", torch.int64, T, c.device),
                                         _vector(outLogProbability, "outLogProbability", torch.float32, T, c.device) if outLogProbability is not None else None),
                "va_sample_in_order")

    def sample(self, logits, uniforms, temperature=1.0, topK=0, topP=1.0, minP=0.0, order: str = "items"):
        """(items, log probabilities)."""
        c, torch = self.context, _torch()
        items, logs = c.empty((logits.shape[0],), torch.int64), c.empty((logits.shape[0],), torch.float32)
        c.order_after_torch()
        self.encode(logits, uniforms, items, logs, temperature, topK, topP, minP, order=order)
        c.synchronize()
        return items, logs
