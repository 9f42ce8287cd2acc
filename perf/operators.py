"""Operators for training and serving an embedding model beside its search index: what is measured.

Three operators that a program with a vector index needs before and after the search itself:

  score / train   softmax cross entropy of hidden rows over all items of a collection (a vocabulary,
                  or the rows of an index): per-row loss and log-sum-exp ("score"), and with them the
                  gradients of the mean loss with respect to the hidden rows and the items ("train")
  codes / norm    root-mean-square norm with the residual's addition: the output in 8 bits with
                  scales ("codes", serving), or in the rows' own type with the backward pass ("norm",
                  training)
  clip            the global 2-norm of a list of gradients, and the gradients clipped by it

Sizes: T rows, V items, D dimensions; "type" is the type of the rows, items and gradients.
"""
from __future__ import annotations

import functools

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_IGNORED = -100
_EPS = 1e-6


def listed():
    return [
        # one interactive query's likelihood over a small collection: nothing but launches and latency
        {"name": "score_1_10k", "kind": "score", "type": "bf16", "T": 1, "V": 10_000, "D": 768, "scale": 20.0, "removed": False},
        # a few queries over a large collection with deleted items, which have no probability: the
        # items are streamed once
        {"name": "score_10_1m", "kind": "score", "type": "f16", "T": 10, "V": 1_000_000, "D": 768, "scale": 20.0, "removed": True},
        # evaluation of a checkpoint in full precision over a collection with no round size
        {"name": "score_512_100k_f32", "kind": "score", "type": "f32", "T": 512, "V": 100_003, "D": 384, "scale": 1.0, "removed": False},
        # one step of tuning a small collection in full precision, a batch of queries
        {"name": "train_100_10k_f32", "kind": "train", "type": "f32", "T": 100, "V": 10_000, "D": 768, "scale": 20.0, "removed": False},
        # an ordinary step, no size round, some rows without a target
        {"name": "train_1023_50k", "kind": "train", "type": "f16", "T": 1023, "V": 49_999, "D": 300, "scale": 1.0, "removed": False},
        # a training step over a large collection, the sampling correction and the deleted items as offsets
        {"name": "train_4096_262k", "kind": "train", "type": "bf16", "T": 4096, "V": 262_144, "D": 768, "scale": 20.0, "removed": True},
        # the last norm of one token, in 8-bit floating point with one scale
        {"name": "codes_1", "kind": "codes", "type": "bf16", "T": 1, "D": 768, "code": "fp8", "group": 0},
        # coding a batch of embeddings as int8 with a scale for each 128 dimensions
        {"name": "codes_64k", "kind": "codes", "type": "bf16", "T": 65_536, "D": 1536, "code": "int8", "group": 128},
        # the norm of a training step, forward and backward, rows that no vector width divides
        {"name": "norm_10k_513", "kind": "norm", "type": "f32", "T": 10_007, "D": 513},
        # the few tensors of a projection head
        {"name": "clip_head", "kind": "clip", "type": "f32", "tensors": 6, "D": 128, "table": 0},
        # the many tensors of an encoder, most of them small
        {"name": "clip_encoder", "kind": "clip", "type": "bf16", "tensors": 290, "D": 384, "table": 0},
        # an encoder's tensors and the table of all items
        {"name": "clip_table", "kind": "clip", "type": "bf16", "tensors": 50, "D": 768, "table": 262_144},
    ]


def _log_int(rng, lo, hi):
    """A whole number whose logarithm is uniform on [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["score", "score", "train", "train", "train", "codes", "codes", "norm", "clip", "clip"])
    kind_type = rng.choice(["f32", "f16", "bf16", "bf16"])
    D = rng.choice([100, 127, 128, 200, 300, 384, 512, 513, 768, 768, 1024, 1536])
    if kind in ("score", "train"):
        T = _log_int(rng, 1, 4096)
        # the largest listed product, 4096 rows by 262,144 items of 768; in full precision a tenth of it
        most = 4096 * 262_144 * 768 // (T * D) // (10 if kind_type == "f32" else 1)
        V = _log_int(rng, 1000, max(1000, min(1_000_000, most, 4096 * 262_144 // T)))
        return {"kind": kind, "type": kind_type, "T": T, "V": V, "D": D, "scale": rng.choice([1.0, 10.0, 20.0]),
                "removed": rng.random() < 0.3}
    if kind == "codes":
        return {"kind": kind, "type": kind_type, "T": _log_int(rng, 1, 65_536), "D": D, "code": rng.choice(["fp8", "int8"]),
                "group": rng.choice([0, 0, 32, 64, 128])}
    if kind == "norm":
        return {"kind": kind, "type": kind_type, "T": _log_int(rng, 1, 65_536), "D": D}
    return {"kind": kind, "type": kind_type, "tensors": _log_int(rng, 1, 400), "D": rng.choice([64, 127, 256, 384, 512, 768]),
            "table": rng.choice([0, 0, _log_int(rng, 1000, 200_000)])}


def _shapes(case):
    """The shapes of a clip case: blocks of square and wide matrices with their vectors, then the table."""
    D = case["D"]
    block = [(D, D), (D,), (D, 4 * D), (4 * D,), (4 * D, D), (D,), (D, D), (D + 1,), (D, D), (3,)]
    shapes = [block[i % len(block)] for i in range(case["tensors"])]
    return shapes + ([(case["table"], D)] if case["table"] else [])


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    kind = case["kind"]
    if kind in ("score", "train"):
        T, V, D = case["T"], case["V"], case["D"]
        items = normal(V, D)
        targets = torch.randint(0, V, (T,), generator=g, device="cuda")
        hidden = normal(T, D)
        if case["scale"] > 1.0:
            # embeddings on the unit sphere, a row near its item; the scale is the inverse temperature
            items /= items.norm(dim=1, keepdim=True)
            hidden = items[targets] + hidden * (1.5 / D**0.5)
            hidden /= hidden.norm(dim=1, keepdim=True)
        else:
            # normalised hidden rows and a projection as it is initialised
            items *= 0.02
        s = {"hidden": hidden.to(dtype), "items": items.to(dtype), "offsets": None}
        if case["removed"]:
            # the correction of items sampled by their frequency; every hundredth or so is deleted
            offsets = -torch.log1p(torch.rand(V, generator=g, device="cuda") * 8.0)
            deleted = torch.rand(V, generator=g, device="cuda") < 0.01
            deleted[targets] = False
            s["offsets"] = offsets.masked_fill(deleted, float("-inf"))
        if kind == "train" and T > 8:
            targets[torch.rand(T, generator=g, device="cuda") < 0.05] = _IGNORED
            targets[0] = V - 1  # one row at least has a target
            if case["removed"]:
                s["offsets"][V - 1] = 0.0
        s |= {"kind": kind, "targets": targets, "scale": case["scale"]}
        f = {"dtype": torch.float32, "device": "cuda"}
        s["out"] = {"loss": torch.empty(T, **f), "lse": torch.empty(T, **f), "mean": torch.empty(1, **f)}
        if kind == "train":
            # the gradient that reaches the mean loss: 1, or a loss scale that keeps half-precision gradients normal
            s["grad"] = torch.full((1,), 16.0 * T if case["type"] == "f16" else 1.0, **f)
            s["out"] |= {"grad_hidden": torch.empty_like(s["hidden"]), "grad_items": torch.empty_like(s["items"])}
        return s
    if kind in ("codes", "norm"):
        T, D = case["T"], case["D"]
        # activations with a few dimensions much larger than the others, as trained encoders have them
        outlier = 1.0 + 9.0 * (torch.rand(D, generator=g, device="cuda") < 0.01)
        s = {"kind": kind, "x": (normal(T, D) * outlier).to(dtype), "residual": (normal(T, D) * 2.0).to(dtype),
             "weight": (1.0 + 0.1 * normal(D)).to(dtype)}
        s["out"] = {"residual": torch.empty_like(s["x"])}
        if kind == "codes":
            groups = -(-D // case["group"]) if case["group"] else 1
            code = torch.int8 if case["code"] == "int8" else torch.float8_e4m3fn
            s |= {"code": case["code"], "group": case["group"]}
            s["codes"] = torch.empty(T, D, dtype=code, device="cuda")
            s["out"]["scales"] = torch.empty(T, groups, dtype=torch.float32, device="cuda")
            # int8 codes are handed back as the values they stand for
            s["out"]["values"] = torch.empty(T, D, dtype=torch.bfloat16, device="cuda") if case["code"] == "int8" else s["codes"]
        else:
            s |= {"grad": normal(T, D).to(dtype), "grad_residual": normal(T, D).to(dtype)}
            s["out"] |= {"y": torch.empty_like(s["x"]), "inverse_rms": torch.empty(T, dtype=torch.float32, device="cuda"),
                         "grad_x": torch.empty_like(s["x"]), "grad_weight": torch.empty_like(s["weight"])}
        return s
    # gradients whose size differs from tensor to tensor
    shapes = _shapes(case)
    sizes = [functools.reduce(lambda a, b: a * b, shape) for shape in shapes]
    flat = torch.empty(sum(sizes), dtype=dtype, device="cuda")
    out = torch.empty_like(flat)
    gradients, outputs, at = [], [], 0
    for i, (shape, n) in enumerate(zip(shapes, sizes)):
        gradients.append(flat[at : at + n].view(shape))
        outputs.append(out[at : at + n].view(shape))
        gradients[-1].copy_(normal(*shape) * (0.001 * (1 + i % 7)))
        at += n
    return {"kind": kind, "gradients": gradients, "outputs": outputs, "flat": out, "max_norm": 1.0,
            "norm": torch.empty(1, dtype=torch.float32, device="cuda")}


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


@functools.lru_cache(maxsize=None)
def _kernels():
    from vectoraccelerate_amd import GPUContext, GradientClipKernel, RMSNormKernel, SoftmaxCrossEntropyKernel

    context = GPUContext(0)
    return SoftmaxCrossEntropyKernel(context), RMSNormKernel(context), GradientClipKernel(context)


def _run_own(s):
    entropy, norm, clip = _kernels()
    kind, out = s["kind"], s.get("out")
    if kind in ("score", "train"):
        entropy.encodeForward(s["hidden"], s["items"], s["targets"], out["loss"], out["lse"], out["mean"], scale=s["scale"],
                              offsets=s["offsets"], ignoreIndex=_IGNORED)
        if kind == "train":
            entropy.encodeBackward(s["hidden"], s["items"], s["targets"], out["lse"], out["grad_hidden"], out["grad_items"],
                                   grad=s["grad"], reduction="mean", scale=s["scale"], offsets=s["offsets"],
                                   ignoreIndex=_IGNORED)
        return out
    if kind == "codes":
        norm.encodeQuantized(s["x"], s["weight"], s["codes"], out["scales"], residual=s["residual"], outResidual=out["residual"],
                             groupSize=s["group"], epsilon=_EPS)
        if s["code"] == "int8":
            norm.encodeDequantize(s["codes"], out["scales"], out["values"], groupSize=s["group"])
        return out
    if kind == "norm":
        norm.encode(s["x"], s["weight"], out["y"], residual=s["residual"], outResidual=out["residual"],
                    outInverseRms=out["inverse_rms"], epsilon=_EPS)
        norm.encodeBackward(s["grad"], out["residual"], s["weight"], out["inverse_rms"], out["grad_x"], out["grad_weight"],
                            gradResidual=s["grad_residual"])
        return out
    if "list" not in s:  # a training program lists its gradients once
        s["list"] = clip.tensorList(s["gradients"], s["outputs"])
    clip.encode(s["list"], s["max_norm"], s["norm"])
    return {"norm": s["norm"], "clipped": s["flat"]}


def _grouped(y, group):
    """y [T, D] as [T, groups, group] (zeros behind the last dimension)."""
    T, D = y.shape
    group = group or D
    return torch.nn.functional.pad(y, (0, -D % group)).view(T, -1, group)


def _run_plain(s):
    kind = s["kind"]
    if kind in ("score", "train"):
        hidden, items, targets = s["hidden"].float(), s["items"].float(), s["targets"]
        logits = (hidden @ items.T) * s["scale"]
        if s["offsets"] is not None:
            logits = logits + s["offsets"]
        counted = targets != _IGNORED
        at = targets.clamp(min=0).unsqueeze(1)
        top = logits.amax(dim=1, keepdim=True)
        lse = top.squeeze(1) + torch.log(torch.exp(logits - top).sum(dim=1))
        loss = torch.where(counted, lse - logits.gather(1, at).squeeze(1), 0.0)
        count = counted.sum().clamp(min=1)
        out = {"loss": loss, "lse": lse, "mean": (loss.sum() / count).view(1)}
        if kind == "train":
            grad = torch.exp(logits - lse.unsqueeze(1))
            grad.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
            grad = grad * (s["grad"] * counted / count).unsqueeze(1)
            out["grad_hidden"] = ((grad @ items) * s["scale"]).to(s["hidden"].dtype)
            out["grad_items"] = ((grad.T @ hidden) * s["scale"]).to(s["items"].dtype)
        return out
    if kind in ("codes", "norm"):
        weight = s["weight"].float()
        r = s["x"].float() + s["residual"].float()
        inverse = torch.rsqrt(r.square().mean(dim=1, keepdim=True) + _EPS)
        y = r * inverse * weight
        residual = r.to(s["x"].dtype)
        if kind == "codes":
            most = 127.0 if s["code"] == "int8" else 448.0
            z = _grouped(y, s["group"])
            scales = z.abs().amax(dim=2, keepdim=True) / most
            z = (z / scales.clamp(min=1e-37)).clamp(-most, most)
            D = y.shape[1]
            if s["code"] == "int8":
                values = (torch.round(z) * scales).view(z.shape[0], -1)[:, :D].to(torch.bfloat16)
            else:
                values = z.view(z.shape[0], -1)[:, :D].to(torch.float8_e4m3fn)
            return {"residual": residual, "scales": scales.squeeze(2), "values": values}
        grad = s["grad"].float()
        kept = residual.float() * inverse
        wg = grad * weight
        grad_x = inverse * (wg - kept * (wg * kept).mean(dim=1, keepdim=True)) + s["grad_residual"].float()
        return {"residual": residual, "y": y.to(s["x"].dtype), "inverse_rms": inverse.squeeze(1), "grad_x": grad_x.to(s["x"].dtype),
                "grad_weight": (grad * kept).sum(dim=0).to(s["weight"].dtype)}
    norm = torch.stack([g.float().square().sum() for g in s["gradients"]]).sum().sqrt()
    factor = (s["max_norm"] / (norm + _EPS)).clamp(max=1.0)
    clipped = torch.cat([(g.float() * factor).to(g.dtype).view(-1) for g in s["gradients"]])
    return {"norm": norm.view(1), "clipped": clipped}


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["type"] == "f32" else 2
    kind = case["kind"]
    if kind in ("score", "train"):
        T, V, D = case["T"], case["V"], case["D"]
        read = size * (T + V) * D + 8 * T + (4 * V if case["removed"] else 0)
        if kind == "score":
            return {"bytes": read + 8 * T + 4, "flops": 2 * T * V * D}
        return {"bytes": read + 8 * T + 4 + size * (T + V) * D, "flops": 6 * T * V * D}
    if kind == "codes":
        T, D = case["T"], case["D"]
        groups = -(-D // case["group"]) if case["group"] else 1
        # x, the residual and the weight; the new residual, the codes and the scales (int8: and the values)
        return {"bytes": T * D * (3 * size + 1 + (2 if case["code"] == "int8" else 0)) + size * D + 4 * T * groups, "flops": 6 * T * D}
    if kind == "norm":
        T, D = case["T"], case["D"]
        # x, the residual and two gradients; the new residual, y and the gradient of x
        return {"bytes": 7 * size * T * D + 2 * size * D + 4 * T, "flops": 14 * T * D}
    n = sum(functools.reduce(lambda a, b: a * b, shape) for shape in _shapes(case))
    return {"bytes": 2 * size * n + 4, "flops": 3 * n}


# ---------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("score", "train"):
        h, w, targets = s["hidden"].double(), s["items"].double(), s["targets"]
        T, V = h.shape[0], w.shape[0]
        counted = torch.nonzero(targets >= 0).flatten()
        count = max(1, counted.numel())
        lse, loss = torch.empty(T, dtype=torch.float64, device="cuda"), torch.zeros(T, dtype=torch.float64, device="cuda")
        gh = torch.zeros_like(h)
        gw = torch.zeros_like(w) if kind == "train" else None
        step = max(1, (1 << 28) // V)
        for t0 in range(0, T, step):
            rows = slice(t0, min(T, t0 + step))
            z = case["scale"] * torch.mm(h[rows], w.t())
            if s["offsets"] is not None:
                z += s["offsets"].double()
            lse[rows] = torch.logsumexp(z, 1)
            here = counted[(counted >= rows.start) & (counted < rows.stop)]
            loss[here] = lse[here] - z[here - t0, targets[here]]
            if kind == "train":
                p = z.sub_(lse[rows, None]).exp_()
                p[here - t0, targets[here]] -= 1.0
                p[targets[rows] < 0] = 0.0
                p *= float(s["grad"]) * case["scale"] / count
                gh[rows] = torch.mm(p, w)
                gw.addmm_(p.t(), h[rows])
            del z
        out = {"loss": loss, "lse": lse, "mean": (loss.sum() / count).view(1)}
        return out | ({"grad_hidden": gh, "grad_items": gw} if kind == "train" else {})
    if kind in ("codes", "norm"):
        w = s["weight"].double()
        D = w.numel()
        r = s["x"].double() + s["residual"].double()
        inverse = 1.0 / torch.sqrt(torch.einsum("td,td->t", r, r) / D + _EPS)
        y = r * inverse[:, None] * w
        if kind == "codes":
            most = 127.0 if case["code"] == "int8" else 448.0
            group = case["group"] or D
            parts = torch.split(y, group, dim=1)
            scales = torch.stack([p.abs().max(dim=1).values / most for p in parts], dim=1)
            z = torch.cat([p / scales[:, i : i + 1] for i, p in enumerate(parts)], dim=1)
            if case["code"] == "int8":
                values = z.round().clamp(-127, 127) * scales.repeat_interleave(group, dim=1)[:, :D]
            else:
                values = z.clamp(-448, 448)
            return {"residual": r, "scales": scales, "values": values}
        # with n = r / rms: dr = (w dy - n mean(w dy n)) / rms, and the residual's own gradient; r as the
        # forward pass stored it
        n = s["x"].float().add(s["residual"].float()).to(s["x"].dtype).double() * inverse[:, None]
        dy = s["grad"].double()
        along = torch.einsum("td,td->t", dy * w, n) / D
        gx = (dy * w - n * along[:, None]) * inverse[:, None] + s["grad_residual"].double()
        return {"residual": r, "y": y, "inverse_rms": inverse, "grad_x": gx, "grad_weight": torch.einsum("td,td->d", dy, n)}
    total = sum(float(g.double().square().sum()) for g in s["gradients"]) ** 0.5
    factor = min(1.0, s["max_norm"] / (total + _EPS))
    return {"norm": torch.tensor([total], dtype=torch.float64), "clipped": torch.cat([g.double().flatten() * factor for g in s["gradients"]])}
