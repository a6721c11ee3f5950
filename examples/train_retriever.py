"""Trains the two sides of a retriever on the GPU and searches with what was trained.

A query is seen through a noisy linear map; its encoder is a projection followed by layer norm, and it is
scored against every row of a table of vectors, one for each item.  A step is

    layer_norm -> softmax_xent_grad -> layer_norm_backward -> orthogonalize (the projection's update)

and the trained table is what CudaKnnEngine then searches, by inner product.  Run it as

    python examples/train_retriever.py [--items 20000] [--dim 128] [--steps 60]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vector-rs_amd"))
import vector_hip as vh  # noqa: E402
from vector_hip import training  # noqa: E402


class Retriever:
    """Encoder x -> layer_norm(x P) and a table of item vectors, trained on softmax cross entropy."""

    def __init__(self, inputs, dim, items, seed=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        make = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
        self.projection = make(inputs, dim) / inputs ** 0.5
        self.momentum = torch.zeros_like(self.projection)
        self.weight, self.bias = torch.ones(dim, device="cuda"), torch.zeros(dim, device="cuda")
        self.table = make(items, dim) / dim ** 0.5

    def encode(self, x):
        return training.layer_norm(x @ self.projection, self.weight, self.bias)[0]

    def step(self, x, item, rate=0.02, table_rate=20.0, beta=0.9):
        """One step on queries x and the items they belong to (negative: padding); the mean loss."""
        z = x @ self.projection
        h, mean, rstd = training.layer_norm(z, self.weight, self.bias)
        counted = (item >= 0).float()
        loss, _, dh, dtable = training.softmax_xent_grad(h, self.table, item, counted / counted.sum())
        dz, dweight, dbias = training.layer_norm_backward(dh, z, self.weight, mean, rstd)
        self.momentum.mul_(beta).add_(x.t() @ dz)
        self.projection -= rate * training.orthogonalize(self.momentum)
        self.weight -= rate * dweight
        self.bias -= rate * dbias
        self.table -= table_rate * dtable
        return loss.sum() / counted.sum()

    def recall(self, x, item, k=10):
        """Share of queries whose item is among the k best of an exact search."""
        engine = vh.CudaKnnEngine(self.table.cpu().numpy(), metric=vh.DistanceMetric.DotProduct)
        ids, _, _ = engine.search_batch_arrays(self.encode(x).cpu().numpy(), k)
        return float((torch.from_numpy(ids.astype("int64")) == item.cpu()[:, None]).any(1).float().mean())


def queries(latent, mix, item, gen):
    """What is seen of items: their latent vector through a linear map, with noise."""
    return latent[item] @ mix + 0.3 * torch.randn(len(item), mix.shape[1], device="cuda", generator=gen)


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--items", type=int, default=20_000)
    p.add_argument("--dim", type=int, default=128)
    p.add_argument("--batch", type=int, default=2048)
    p.add_argument("--steps", type=int, default=60)
    a = p.parse_args(argv)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    latent = torch.randn(a.items, 32, device="cuda", generator=gen)
    mix = torch.randn(32, 96, device="cuda", generator=gen) / 32 ** 0.5
    model = Retriever(96, a.dim, a.items)
    held = torch.randint(0, a.items, (1000,), device="cuda", generator=gen)
    seen = queries(latent, mix, held, gen)
    before = model.recall(seen, held)
    first = last = None
    for step in range(a.steps):
        item = torch.randint(0, a.items, (a.batch,), device="cuda", generator=gen)
        loss = model.step(queries(latent, mix, item, gen), item)
        if step % 20 == 0 or step + 1 == a.steps:
            last = float(loss)
            first = last if first is None else first
            print(f"step {step:4d}  loss {last:.3f}", flush=True)
    after = model.recall(seen, held)
    print(f"recall@10 over {a.items} items: {before:.3f} before, {after:.3f} after")
    return first, last, before, after


if __name__ == "__main__":
    main()
