"""Train the embeddings of a collection, code them in 8 bits and search them.

    python examples/train_and_serve.py [--items 20000] [--dim 128] [--steps 60]

Every item has a hidden prototype that only its queries' features (noisy copies) show.  The encoder is
one linear layer with a residual and an RMS norm; the loss is the softmax cross entropy of the encoded
query over all items (an item in use is one of the vocabulary, a deleted one is masked):

    r = x + x P      h = r / rms(r) * w      l = scale * h . items + offsets

A step runs the norm forward, the loss and its gradients, the norm backward, and clips all gradients
together before they are taken.  Afterwards queries are normalised straight into int8 codes on the grid of
one given scale, the items are coded on theirs, and the int8 scan finds each query's items.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from vectoraccelerate_amd import (GPUContext, GradientClipKernel, PerDimensionParameters, RMSNormKernel, ScalarQuantizationKernel,  # noqa: E402
                                  SoftmaxCrossEntropyKernel)


class Encoder:
    """Parameters and the two directions of h = norm(x + x P) * w."""

    def __init__(self, context: GPUContext, dim: int, dtype, generator):
        self.norm = RMSNormKernel(context)
        self.P = (torch.randn(dim, dim, device="cuda", generator=generator) * 0.1 / dim**0.5).to(dtype)
        self.w = torch.ones(dim, device="cuda", dtype=dtype)

    def forward(self, x):
        h, r, inverse = self.norm.forward(x @ self.P, self.w, x)
        return h, (x, r, inverse)

    def backward(self, grad, saved):
        x, r, inverse = saved
        gr, gw = self.norm.backward(grad, r, self.w, inverse)
        return x.T @ gr, gw

    def codes(self, x, scale: float):
        """int8 codes of the encoded rows on one grid, as the int8 scan compares them."""
        return self.norm.quantize(x @ self.P, self.w, x, torch.int8, givenScale=scale)[0]


def queries_of(prototypes, targets, generator):
    return prototypes[targets] + 0.5 * torch.randn(targets.numel(), prototypes.shape[1], device="cuda", generator=generator).to(prototypes.dtype)


def run(context: GPUContext, items: int = 20_000, dim: int = 128, batch: int = 1024, steps: int = 60, dtype=torch.float32, rate: float = 0.1,
        seed: int = 0) -> dict:
    g = torch.Generator("cuda").manual_seed(seed)
    entropy, clip, scan = SoftmaxCrossEntropyKernel(context), GradientClipKernel(context), ScalarQuantizationKernel(context)
    prototypes = torch.randn(items, dim, device="cuda", generator=g).to(dtype)
    table = (0.1 * torch.randn(items, dim, device="cuda", generator=g)).to(dtype)
    offsets = torch.zeros(items, device="cuda")
    deleted = torch.randperm(items, device="cuda", generator=g)[: items // 50]
    offsets[deleted] = -torch.inf
    live = torch.nonzero(offsets == 0).squeeze(1)
    encoder, scale = Encoder(context, dim, dtype, g), dim**-0.5
    parameters = [table, encoder.P, encoder.w]
    optimizer = torch.optim.Adam([{"params": [table], "lr": rate}, {"params": [encoder.P, encoder.w], "lr": 0.03 * rate}], betas=(0.9, 0.99))

    losses, norms = [], []
    for _ in range(steps):
        y = live[torch.randint(0, live.numel(), (batch,), device="cuda", generator=g)]
        h, saved = encoder.forward(queries_of(prototypes, y, g))
        out = entropy.forward(h, table, y, "mean", scale, offsets)
        grad_h, grad_table = entropy.backward(h, table, y, out.logSumExp, None, "mean", scale, offsets)
        grad_P, grad_w = encoder.backward(grad_h, saved)
        gradients = [grad_table, grad_P, grad_w]
        norms.append(clip.clip(gradients, 0.2))
        for p, d in zip(parameters, gradients):
            p.grad = d
        optimizer.step()
        losses.append(float(out.reduced))

    # serving: deleted items leave the collection, both sides are coded on one grid each
    kept = table[live].float()
    step = torch.tensor([float(kept.abs().max()) / 127.0] * dim).numpy()
    grid = PerDimensionParameters(-127 * step, 127 * step, step, np.zeros(dim, np.int32))
    item_codes = scan.quantizePerDimension(kept.contiguous(), grid)
    y = torch.randint(0, live.numel(), (512,), device="cuda", generator=g)
    x = queries_of(prototypes, live[y], g)
    h, _ = encoder.forward(x)
    found, _ = scan.searchTopK(encoder.codes(x, float(h.abs().max()) / 127.0), item_codes, 10)
    exact = (h.float() @ kept.T).topk(10, 1).indices.cpu().numpy()
    same = np.mean([len(set(a) & set(b)) / 10 for a, b in zip(found.tolist(), exact.tolist())])
    hit = (found == y.cpu().numpy()[:, None]).any(1).mean()
    return {"losses": losses, "norms": norms, "top10_agreement": float(same), "target_in_top10": float(hit)}


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--items", type=int, default=20_000)
    p.add_argument("--dim", type=int, default=128)
    p.add_argument("--batch", type=int, default=1024)
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--dtype", choices=["float32", "float16", "bfloat16"], default="float32")
    a = p.parse_args()
    r = run(GPUContext(0), a.items, a.dim, a.batch, a.steps, getattr(torch, a.dtype))
    for i in range(0, a.steps, max(1, a.steps // 8)):
        print(f"step {i:4d}  loss {r['losses'][i]:.4f}  gradient norm {r['norms'][i]:.4f}")
    print(f"last       loss {r['losses'][-1]:.4f}")
    print(f"int8 top 10 agrees with the exact one in {100 * r['top10_agreement']:.1f} %; holds the target of {100 * r['target_in_top10']:.1f} % of the queries")


if __name__ == "__main__":
    main()
