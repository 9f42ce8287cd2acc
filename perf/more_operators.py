"""Operators for training a collection's embeddings, keeping them in 4 bits and answering with them: what is measured.

Three operators next to the loss, the norm and the clipping of perf/operators.py:

  adamw           one AdamW step over a list of tensors, its moments in 32 bits or in 8, gradients clipped by a
                  norm that the program has already ("masters": the parameters' 32-bit copies)
  quant / score   rows in microscaled 4-bit floating point (e2m1 in blocks of 32 with a power of two each): coding
                  and reading back, and the product of queries with all items of a collection; the queries are
                  coded in the call ("mx") or stay in 16 bits ("plain")
  sample          an item for each row of logits, by temperature, top-k, top-p and min-p, from a given random number

Sizes: T rows, V items, D dimensions; "type" is the type of the parameters, rows or logits.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BETA1, _BETA2, _EPS = 0.9, 0.999, 1e-8
_RATE, _DECAY, _STEP, _SEED = 1e-3, 0.01, 100, 7
_GROUP = 256  # values of an 8-bit moment that share a scale; a tensor's first value starts one


def listed():
    return [
        # the few tensors of a projection head, full precision: nothing but the call and one launch
        {"name": "adamw_head", "kind": "adamw", "type": "f32", "bits": 32, "masters": False, "clip": False, "tensors": 6, "D": 128, "table": 0},
        # the many tensors of an encoder in bf16 with 32-bit copies, clipped by the norm of all gradients
        {"name": "adamw_encoder", "kind": "adamw", "type": "bf16", "bits": 32, "masters": True, "clip": True, "tensors": 290, "D": 384, "table": 0},
        # an encoder's tensors and the table of all items, moments in 8 bits so that the table's fit
        {"name": "adamw_table_8bit", "kind": "adamw", "type": "bf16", "bits": 8, "masters": False, "clip": True, "tensors": 50, "D": 768, "table": 262_144},
        # coding a batch of embeddings as it enters the collection, and reading it back
        {"name": "quant_64k", "kind": "quant", "type": "bf16", "T": 65_536, "D": 1536},
        # one interactive query against a small collection: launches and latency
        {"name": "score_1_10k", "kind": "score", "type": "bf16", "queries": "plain", "out": "f32", "T": 1, "V": 10_000, "D": 768, "removed": False},
        # a few queries against a large collection with deleted items: its codes are streamed once
        {"name": "score_10_1m", "kind": "score", "type": "f16", "queries": "plain", "out": "f32", "T": 10, "V": 1_000_000, "D": 768, "removed": True},
        # an evaluation's queries, coded on the way, no size round, scores in full precision
        {"name": "score_512_100k", "kind": "score", "type": "f32", "queries": "mx", "out": "f32", "T": 512, "V": 100_003, "D": 384, "removed": False},
        # a large batch against a large collection, logits in 16 bits
        {"name": "score_4096_262k", "kind": "score", "type": "bf16", "queries": "mx", "out": "bf16", "T": 4096, "V": 262_144, "D": 768, "removed": False},
        # one interactive row
        {"name": "sample_1_10k", "kind": "sample", "type": "f32", "T": 1, "V": 10_000, "spread": 2.0, "temperature": 0.8, "k": 50, "p": 0.95, "m": 0.0, "mixed": False, "removed": False},
        # a batch in service over a long axis, by its nucleus
        {"name": "sample_64_262k", "kind": "sample", "type": "bf16", "T": 64, "V": 262_144, "spread": 2.5, "temperature": 0.7, "k": 0, "p": 0.9, "m": 0.02, "mixed": False, "removed": False},
        # a batch whose rows each have settings of their own, some of them greedy, deleted items masked
        {"name": "sample_512_50k_mixed", "kind": "sample", "type": "f32", "T": 512, "V": 49_999, "spread": 2.0, "temperature": 1.0, "k": 0, "p": 1.0, "m": 0.0, "mixed": True, "removed": True},
        # negatives for training, drawn from the whole softmax
        {"name": "sample_2048_100k", "kind": "sample", "type": "f16", "T": 2048, "V": 100_003, "spread": 1.0, "temperature": 1.0, "k": 0, "p": 1.0, "m": 0.0, "mixed": False, "removed": False},
    ]


def _log_int(rng, lo, hi):
    """A whole number whose logarithm is uniform on [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["adamw", "adamw", "quant", "score", "score", "score", "sample", "sample", "sample"])
    of = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "adamw":
        return {"kind": kind, "type": of, "bits": rng.choice([8, 32]), "masters": of != "f32" and rng.random() < 0.5, "clip": rng.random() < 0.5,
                "tensors": _log_int(rng, 1, 300), "D": rng.choice([64, 127, 256, 384, 512]), "table": rng.choice([0, 0, _log_int(rng, 1000, 200_000)])}
    D = rng.choice([100, 127, 128, 200, 300, 384, 512, 513, 768, 768, 1024, 1536])
    if kind == "quant":
        return {"kind": kind, "type": of, "T": _log_int(rng, 1, 65_536), "D": D}
    T = _log_int(rng, 1, 4096)
    if kind == "score":
        queries = "mx" if of == "f32" else rng.choice(["mx", "plain"])
        # the largest listed product; queries in 16 bits, which serve few rows, a quarter of it
        most = 4096 * 262_144 * 768 // (T * D) // (4 if queries == "plain" else 1)
        V = _log_int(rng, 1000, max(1000, min(1_000_000, most, 4096 * 262_144 // T // 2, 1_000_000 * 768 // D)))
        return {"kind": kind, "type": of, "queries": queries, "out": rng.choice(["f32", "f16", "bf16"]), "T": T, "V": V, "D": D, "removed": rng.random() < 0.3}
    V = _log_int(rng, 1000, max(1000, min(1_000_000, 2048 * 100_003 // T)))
    return {"kind": kind, "type": of, "T": T, "V": V, "spread": rng.choice([0.3, 1.0, 2.0, 3.0]), "temperature": rng.choice([0.5, 0.8, 1.0, 1.5]),
            "k": rng.choice([0, 0, _log_int(rng, 1, 1000)]), "p": rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]), "m": rng.choice([0.0, 0.0, 0.01, 0.1]),
            "mixed": rng.random() < 0.3, "removed": rng.random() < 0.3}


def _shapes(case):
    """The shapes of an adamw case: blocks of square and wide matrices with their vectors, then the table."""
    D = case["D"]
    block = [(D, D), (D,), (D, 3 * D), (3 * D,), (3 * D, D), (D,), (D, D), (D + 1,), (D, D), (3,)]
    shapes = [block[i % len(block)] for i in range(case["tensors"])]
    return shapes + ([(case["table"], D)] if case["table"] else [])


def _size(shape):
    return functools.reduce(lambda a, b: a * b, shape)


def _padded(n):
    return -(-n // _GROUP) * _GROUP


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    kind = case["kind"]
    if kind == "adamw":
        # the tensors lie one behind another, each from a multiple of 256 values on
        shapes = _shapes(case)
        sizes = [_size(shape) for shape in shapes]
        starts, at = [], 0
        for n in sizes:
            starts.append(at)
            at += _padded(n)
        there = torch.zeros(at, dtype=torch.bool, device="cuda")
        for a, n in zip(starts, sizes):
            there[a : a + n] = True
        size_of = torch.tensor([0.2 + 0.3 * (i % 7) for i in range(len(sizes))], device="cuda")
        size_of = size_of.repeat_interleave(torch.tensor([_padded(n) for n in sizes], device="cuda"), output_size=at)
        grad = normal(at) * size_of * there * 1e-3
        # a hundred steps in: the moments of gradients like these
        first = (grad * 0.3 + normal(at) * size_of * 2e-4) * there
        second = (size_of * 1e-3).square() * (0.1 * (0.5 + torch.rand(at, generator=g, device="cuda"))) * there
        param = normal(at) * 0.02 * there
        now = {"parameters": param.to(dtype)}
        if case["masters"]:
            now["masters"] = param
        if case["bits"] == 8:
            for name, x in (("first", first), ("second", second.sqrt())):
                top = x.view(-1, _GROUP).abs().amax(dim=1)
                now[name + "_scales"] = top / 448.0
                now[name] = (x.view(-1, _GROUP) / (top / 448.0).clamp(min=1e-30).unsqueeze(1)).clamp(-448, 448).view(-1).to(torch.float8_e4m3fn)
        else:
            now |= {"first": first, "second": second}
        s = {"kind": kind, "bits": case["bits"], "sizes": sizes, "starts": starts, "gradients": grad.to(dtype), "now": now,
             "next": {k: torch.zeros_like(v) for k, v in now.items()},
             # vectors (the norms' weights, the biases) do not decay
             "decays": [0.0 if len(shape) == 1 else 1.0 for shape in shapes], "norm": None}
        if case["clip"]:
            s["norm"] = s["gradients"].float().square().sum().sqrt().view(1)
            s["max_norm"] = float(s["norm"]) / 1.7
        return s
    if kind == "quant":
        T, D = case["T"], case["D"]
        outlier = 1.0 + 9.0 * (torch.rand(D, generator=g, device="cuda") < 0.01)
        s = {"kind": kind, "x": (normal(T, D) * outlier).to(dtype)}
        s["out"] = _empty_codes(T, D) | {"values": torch.empty(T, D, dtype=torch.bfloat16, device="cuda")}
        return s
    if kind == "score":
        T, V, D = case["T"], case["V"], case["D"]
        items = normal(V, D)
        items /= items.norm(dim=1, keepdim=True)
        near = torch.randint(0, V, (T,), generator=g, device="cuda")
        x = items[near] + normal(T, D) * (1.5 / D**0.5)
        x /= x.norm(dim=1, keepdim=True)
        codes, scales = _code(items)
        s = {"kind": kind, "queries": case["queries"], "x": x.to(dtype), "codes": codes, "scales": scales, "scale": 20.0, "offsets": None}
        if case["removed"]:
            offsets = -torch.log1p(torch.rand(V, generator=g, device="cuda") * 8.0)
            s["offsets"] = offsets.masked_fill(torch.rand(V, generator=g, device="cuda") < 0.01, float("-inf"))
        if case["queries"] == "mx":
            s["coded"] = _empty_codes(T, D)
        s["out"] = torch.empty(T, V, dtype=_TYPES[case["out"]], device="cuda")
        return s
    T, V = case["T"], case["V"]
    logits = normal(T, V) * case["spread"]
    # a few items are far more likely than the others
    peaks = torch.randint(0, V, (T, 20), generator=g, device="cuda")
    logits.scatter_add_(1, peaks, (2.0 + normal(T, 20).abs()) * case["spread"])
    if case["removed"]:
        logits.masked_fill_(torch.rand(V, generator=g, device="cuda") < 0.01, float("-inf"))
    s = {"kind": kind, "logits": logits.to(dtype), "uniforms": torch.rand(T, generator=g, device="cuda")}
    if case["mixed"]:
        def among(values, of):
            return torch.tensor(values, dtype=of, device="cuda")[torch.randint(0, len(values), (T,), generator=g, device="cuda")]

        s["set"] = {"temperature": among([0.0, 0.6, 0.8, 1.0, 1.3], torch.float32), "topK": among([0, 0, 1, 20, 50, 400], torch.int32),
                    "topP": among([1.0, 0.8, 0.9, 0.95], torch.float32), "minP": among([0.0, 0.0, 0.05], torch.float32)}
    else:
        s["set"] = {"temperature": case["temperature"], "topK": case["k"], "topP": case["p"], "minP": case["m"]}
    s["out"] = {"items": torch.empty(T, dtype=torch.int64, device="cuda"), "log_probability": torch.empty(T, dtype=torch.float32, device="cuda")}
    return s


def _empty_codes(T, D):
    """Rows in 4 bits: padded to whole groups of 128 values, 64 bytes of codes and 4 of scales each."""
    groups = -(-D // 128)
    return {"codes": torch.empty(T, 64 * groups, dtype=torch.uint8, device="cuda"), "scales": torch.empty(T, 4 * groups, dtype=torch.uint8, device="cuda")}


def _code(x):
    """Codes (two a byte, the even dimension in the low half) and scale bytes of fp32 rows."""
    T, D = x.shape
    x = torch.nn.functional.pad(x, (0, -D % 128)).view(T, -1, 32)
    top = x.abs().amax(dim=2, keepdim=True)
    exponent = torch.frexp(top).exponent - 1  # top = 2^exponent (1 to 2)
    # the least power of two with which no value rounds past 6, the largest that e2m1 has
    exponent = (exponent - 2 + (torch.ldexp(top, 2 - exponent) >= 7.0)).clamp(min=-127)
    exponent = torch.where(top == 0, -127, exponent)
    a = torch.ldexp(x.abs(), (-exponent).clamp(max=120)) * torch.exp2((-exponent - 120).clamp(min=0).float())
    a = torch.where(a < 2, torch.round(2 * a), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4)).clamp(max=7)
    nibble = (a + 8 * torch.signbit(x)).to(torch.uint8).view(T, -1)
    return nibble[:, 0::2] | nibble[:, 1::2] << 4, (exponent.squeeze(2) + 127).to(torch.uint8)


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


@functools.lru_cache(maxsize=None)
def _kernels():
    from vectoraccelerate_amd import AdamWKernel, GPUContext, MicroscaledQuantizationKernel, SoftmaxSamplingKernel

    context = GPUContext(0)
    return AdamWKernel(context), MicroscaledQuantizationKernel(context), SoftmaxSamplingKernel(context)


def _state_of(s, buffers):
    """The framework's lists of a program's tensors: (parameters, state)."""
    from vectoraccelerate_amd import AdamWState

    def cut(name, per=1):
        if name not in buffers:
            return None
        return [buffers[name][a // per : a // per - (-n // per)] for a, n in zip(s["starts"], s["sizes"])]

    return cut("parameters"), AdamWState(cut("first"), cut("second"), cut("first_scales", _GROUP), cut("second_scales", _GROUP), cut("masters"))


def _run_own(s):
    adamw, microscaled, sampling = _kernels()
    kind = s["kind"]
    if kind == "adamw":
        if "list" not in s:  # a training program lists its tensors once
            gradients = [s["gradients"][a : a + n] for a, n in zip(s["starts"], s["sizes"])]
            parameters, state = _state_of(s, s["now"])
            s["list"] = adamw.tensorList(parameters, gradients, state, outputs=_state_of(s, s["next"]), decayFactors=s["decays"])
        adamw.encode(s["list"], _STEP, _RATE, _BETA1, _BETA2, _EPS, _DECAY, gradNorm=s["norm"], maxNorm=s.get("max_norm"), seed=_SEED)
        return s["next"]
    from vectoraccelerate_amd import MicroscaledRows

    if kind == "quant":
        out, x = s["out"], s["x"]
        rows = MicroscaledRows(out["codes"], out["scales"], x.shape[1])
        microscaled.encodeQuantize(x, rows)
        microscaled.encodeDequantize(rows, out["values"])
        return {"scales": out["scales"], "values": out["values"]}
    if kind == "score":
        D = s["x"].shape[1]
        queries = s["x"]
        if s["queries"] == "mx":
            queries = MicroscaledRows(s["coded"]["codes"], s["coded"]["scales"], D)
            microscaled.encodeQuantize(s["x"], queries)
        microscaled.encodeProduct(queries, MicroscaledRows(s["codes"], s["scales"], D), s["out"], scale=s["scale"], offsets=s["offsets"])
        return s["out"]
    sampling.encode(s["logits"], s["uniforms"], s["out"]["items"], s["out"]["log_probability"], **s["set"], order="logits")
    return s["out"]


def _values(codes, scales, D):
    """The fp32 rows that 4-bit codes and their scale bytes stand for."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device="cuda")
    pairs = torch.stack([codes & 15, codes >> 4], dim=2).view(codes.shape[0], -1, 32)
    return torch.ldexp(grid[pairs.int()], scales.int().unsqueeze(2) - 127).view(codes.shape[0], -1)[:, :D]


def _mixed(z):
    """splitmix64's output function; the shifts are of the unsigned word."""
    z = (z ^ ((z >> 30) & ((1 << 34) - 1))) * -0x40A7B892E31B1A47
    z = (z ^ ((z >> 27) & ((1 << 37) - 1))) * -0x6B2FB644ECCEEE15
    return z ^ ((z >> 31) & ((1 << 33) - 1))


def _randoms(count):
    """16 random bits for each value of the first moment and each of the second: a word for each pair of values."""
    golden = -0x61C8864680B583EB
    base = _mixed(golden * torch.tensor(_STEP, device="cuda") + _SEED)
    z = _mixed(base + golden * torch.arange(1, count // 2 + 1, device="cuda"))
    halves = torch.stack([z & 0xFFFF, (z >> 16) & 0xFFFF, (z >> 32) & 0xFFFF, (z >> 48) & 0xFFFF], dim=1).view(-1, 2).float()
    return halves[:, 0], halves[:, 1]


def _coded(x, random, least):
    """e4m3 codes and scales of groups of 256, rounded up with the probability of the part cut off."""
    x = x.view(-1, _GROUP)
    top = x.abs().amax(dim=1, keepdim=True)
    top = torch.where(top < 2.0**-100, 0.0, top)
    z = (x.abs() * torch.where(top > 0, 448.0 / top, 0.0)).clamp(max=448.0)
    step = torch.exp2((torch.frexp(z).exponent - 1).clamp(min=-6).float() - 3)
    z = (torch.floor(z / step + random.view(-1, _GROUP) / 65536) * step).clamp(max=448.0)
    if least:  # what is not zero stays so
        z = torch.where((x > 0) & (top > 0) & (z == 0), 2.0**-9, z)
    return torch.copysign(z, x).view(-1).to(torch.float8_e4m3fn), (top / 448.0).view(-1)


def _run_plain(s):
    kind = s["kind"]
    if kind == "adamw":
        now, padded = s["now"], [_padded(n) for n in s["sizes"]]
        total = sum(padded)
        grad = s["gradients"].float()
        if s["norm"] is not None:
            grad = grad * (s["max_norm"] / (s["norm"] + 1e-6)).clamp(max=1.0)
        first, second = now["first"].float(), now["second"].float()
        if s["bits"] == 8:
            first = (first.view(-1, _GROUP) * now["first_scales"].unsqueeze(1)).view(-1)
            second = (second.view(-1, _GROUP) * now["second_scales"].unsqueeze(1)).view(-1).square()
        first = _BETA1 * first + (1.0 - _BETA1) * grad
        second = _BETA2 * second + (1.0 - _BETA2) * grad.square()
        decay = torch.tensor(s["decays"], device="cuda").repeat_interleave(torch.tensor(padded, device="cuda"), output_size=total)
        param = now["masters"] if "masters" in now else now["parameters"].float()
        root = second.sqrt()
        moved = first / (root / math.sqrt(1.0 - _BETA2**_STEP) + _EPS)
        param = param * (1.0 - (_RATE * _DECAY) * decay) - (_RATE / (1.0 - _BETA1**_STEP)) * moved
        out = {"parameters": param.to(now["parameters"].dtype)}
        if "masters" in now:
            out["masters"] = param
        if s["bits"] == 8:
            for_first, for_second = _randoms(total)
            out["first"], out["first_scales"] = _coded(first, for_first, False)
            out["second"], out["second_scales"] = _coded(root, for_second, True)
            return out
        return out | {"first": first, "second": second}
    if kind == "quant":
        codes, scales = _code(s["x"].float())
        return {"scales": scales, "values": _values(codes, scales, s["x"].shape[1]).to(torch.bfloat16)}
    if kind == "score":
        D = s["x"].shape[1]
        x = s["x"].float()
        if s["queries"] == "mx":
            x = _values(*_code(x), D)
        scores = (x @ _values(s["codes"], s["scales"], D).T) * s["scale"]
        if s["offsets"] is not None:
            scores = scores + s["offsets"]
        return scores.to(s["out"].dtype)
    x, u, settings = s["logits"], s["uniforms"], s["set"]
    T, V = x.shape

    def column(v):
        return v.double().view(T, 1) if isinstance(v, torch.Tensor) else torch.full((T, 1), v, dtype=torch.float32, device="cuda").double()

    temperature, k, p, m = (column(settings[name]) for name in ("temperature", "topK", "topP", "minP"))
    k = torch.where(temperature == 0, 1, torch.where(k == 0, V, k))
    # ties are in the order of their items; 64 bits: a draw next to a border falls on its side of it
    x, order = torch.sort(x.float(), dim=1, descending=True, stable=True)
    x = x.double()
    w = torch.exp((x - x[:, :1]) / torch.where(temperature == 0, 1, temperature))
    upto = w.cumsum(dim=1)
    before = torch.nn.functional.pad(upto[:, :-1], (1, 0))
    keep = torch.arange(V, device="cuda") < k
    total = (w * keep).sum(dim=1, keepdim=True)
    keep &= (before < p * total) & (w >= m)
    total = upto.gather(1, keep.sum(dim=1, keepdim=True) - 1)
    at = ((upto <= u.double().view(T, 1) * total) & keep).sum(dim=1, keepdim=True).minimum(keep.sum(dim=1, keepdim=True) - 1)
    return {"items": order.gather(1, at).view(T), "log_probability": torch.log(w.gather(1, at) / total).float().view(T)}


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["type"] == "f32" else 2
    kind = case["kind"]
    if kind == "adamw":
        n = sum(_size(shape) for shape in _shapes(case))
        moments = 2 * (1 + 4 / _GROUP) if case["bits"] == 8 else 8
        # gradients; the moments and the parameters in and out (of parameters with a 32-bit copy, the copy in and both out)
        return {"bytes": n * (size + 2 * moments + (8 + size if case["masters"] else 2 * size)), "flops": 14 * n}
    if kind == "quant":
        T, D = case["T"], case["D"]
        return {"bytes": T * D * (size + 2) + T * (D / 2 + D / 32) * 2, "flops": 6 * T * D}
    if kind == "score":
        T, V, D = case["T"], case["V"], case["D"]
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": V * (D / 2 + D / 32) + size * T * D + out * T * V + (4 * V if case["removed"] else 0), "flops": 2 * T * V * D}
    T, V = case["T"], case["V"]
    return {"bytes": size * T * V + 16 * T, "flops": 6 * T * V}


# ---------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "adamw":
        return _exact_adamw(s, case)
    if kind == "quant":
        values, exponents = _exact_code(s["x"].double())
        return {"scales": None, "values": values}
    if kind == "score":
        D = case["D"]
        x = s["x"].double()
        if case["queries"] == "mx":
            x = _exact_code(x)[0]
        out = torch.empty(case["T"], case["V"], dtype=torch.float64, device="cuda")
        low, high = (torch.bitwise_right_shift(s["codes"], n).bitwise_and(15).long() for n in (0, 4))
        step = max(1, (1 << 27) // D)
        for v in range(0, case["V"], step):
            rows = slice(v, min(case["V"], v + step))
            w = torch.empty(rows.stop - v, 2 * low.shape[1], dtype=torch.float64, device="cuda")
            for at, half in ((0, low), (1, high)):
                e, f = half[rows] % 8 // 2, half[rows] % 2  # exponent and fraction bit of e2m1
                a = torch.where(e == 0, 0.5 * f, torch.pow(2.0, (e - 1).double()) * (1 + 0.5 * f))
                w[:, at::2] = torch.where(half[rows] >= 8, -a, a)
            w *= torch.pow(2.0, s["scales"][rows].double() - 127).repeat_interleave(32, dim=1)
            out[:, rows] = torch.mm(x, w[:, :D].t()) * 20.0
        return out if s["offsets"] is None else out.add_(s["offsets"].double())
    items, logs, u = [], [], s["uniforms"].double()
    T, V = s["logits"].shape
    step = max(1, (1 << 26) // V)
    for t in range(0, T, step):
        rows = slice(t, min(T, t + step))
        x = s["logits"][rows].double()
        n = x.shape[0]
        setting = [torch.as_tensor(s["set"][name], device="cuda")[rows].double() if case["mixed"] else
                   torch.full((n,), s["set"][name], dtype=torch.float32, device="cuda").double() for name in ("temperature", "topK", "topP", "minP")]
        greedy = setting[0] == 0
        k = torch.where(greedy, 1, torch.where(setting[1] == 0, V, setting[1])).long()
        order = torch.argsort(-x, dim=1, stable=True)
        probability = torch.softmax(torch.gather(x, 1, order) / torch.where(greedy, 1, setting[0])[:, None], dim=1)
        cumulated = torch.cumsum(probability, 1)
        all_k = cumulated.gather(1, k[:, None] - 1)
        # the nucleus ends with the first item that brings the sum to p; min-p and top-k may end it before
        kept = torch.searchsorted(cumulated, setting[2][:, None] * all_k).squeeze(1) + 1
        kept = torch.where(setting[2] >= 1, V, kept).minimum(k).minimum((probability >= setting[3][:, None] * probability[:, :1]).sum(1))
        all_kept = cumulated.gather(1, kept[:, None] - 1)
        at = torch.searchsorted(cumulated, u[rows, None] * all_kept, right=True).squeeze(1).minimum(kept - 1)[:, None]
        items.append(order.gather(1, at).squeeze(1))
        logs.append((probability.gather(1, at) / all_kept).log().squeeze(1))
    return {"items": torch.cat(items), "log_probability": torch.cat(logs)}


def _exact_code(x):
    """(the values that rows in 64 bits are coded as, the blocks' exponents), by distances to all e2m1 values."""
    T, D = x.shape
    values, exponents = torch.empty_like(x), []
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    for d in range(0, D, 32):
        part = x[:, d : d + 32]
        top = part.abs().max(dim=1, keepdim=True).values
        exponent = torch.floor(torch.log2(top / 7.0)) + 1  # top < 7 2^exponent
        exponent = torch.where(top >= 7 * torch.pow(2.0, exponent), exponent + 1, exponent)
        exponent = torch.where(top < 7 * torch.pow(2.0, exponent - 1), exponent - 1, exponent)
        exponent = torch.where(top == 0, -127.0, exponent).clamp(min=-127)
        a = part.abs() / torch.pow(2.0, exponent)
        best = torch.zeros_like(a)
        far = a.clone()
        for code in range(1, 8):
            d_code = (a - grid[code]).abs()
            nearer = (d_code < far) | ((d_code == far) & (code % 2 == 0))
            best, far = torch.where(nearer, grid[code], best), torch.where(nearer, d_code, far)
        values[:, d : d + 32] = torch.copysign(best * torch.pow(2.0, exponent), part)
        exponents.append(exponent)
    return values, torch.cat(exponents, dim=1)


def _exact_adamw(s, case):
    now, total = s["now"], s["gradients"].numel()
    g = s["gradients"].double()
    if case["clip"]:
        g = g * min(1.0, s["max_norm"] / (float(s["norm"]) + 1e-6))
    m, v = now["first"].double(), now["second"].double()
    if case["bits"] == 8:
        m = m * now["first_scales"].double().repeat_interleave(_GROUP)
        v = (v * now["second_scales"].double().repeat_interleave(_GROUP)) ** 2
    m = m + (1 - _BETA1) * (g - m)
    v = v + (1 - _BETA2) * (g * g - v)
    p = now.get("masters", now["parameters"]).double()
    decay = torch.zeros(total, dtype=torch.float64, device="cuda")
    for a, n, f in zip(s["starts"], s["sizes"], s["decays"]):
        decay[a : a + n] = f * _DECAY
    p = p - _RATE * (decay * p + m / (1 - _BETA1**_STEP) / (torch.sqrt(v / (1 - _BETA2**_STEP)) + _EPS))
    out = {"parameters": p, "masters": p if case["masters"] else None, "first": m, "second": v}
    if case["bits"] == 8:
        # a code is one of the two e4m3 values around the quotient, by chance: the scales alone have one value
        tops = {name: x.view(-1, _GROUP).abs().max(dim=1).values / 448.0 for name, x in (("first", m), ("second", v.sqrt()))}
        out |= {"first": None, "second": None, "first_scales": tops["first"], "second_scales": tops["second"]}
    return {k: x for k, x in out.items() if x is not None or k in now}
