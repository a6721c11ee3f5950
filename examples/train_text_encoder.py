"""Trains a small text encoder on the GPU and searches with what it makes of texts.

A text is a run of words about a topic; texts of different lengths lie one after the other in one array.  Words have
vectors, one layer of causal attention with grouped heads mixes them, and a text is what its last word has become.  A step is

    words -> qk_norm_rotary -> attention -> layer_norm -> softmax_xent_grad (against a vector for each topic)
    -> layer_norm_backward -> attention_backward -> qk_norm_rotary_backward -> clip_gradients -> orthogonalize

and CudaKnnEngine then finds a text's nearest ones by inner product.  Run it as

    python examples/train_text_encoder.py [--topics 200] [--steps 80]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vector-rs_amd"))
import vector_hip as vh  # noqa: E402
from vector_hip import training  # noqa: E402


class TextEncoder:
    """Word vectors, one layer of attention over them, and a vector for each topic."""

    def __init__(self, words, topics, dim=64, heads=4, kv_heads=2, seed=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        make = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
        self.heads, self.kv_heads, self.size = heads, kv_heads, dim // heads
        inner = (heads + 2 * kv_heads) * self.size
        self.weights = {
            "words": make(words, dim) / dim ** 0.5,
            "qkv": make(dim, inner) / dim ** 0.5,
            "out": make(heads * self.size, dim) / dim ** 0.5,
            "q": torch.ones(self.size, device="cuda"),
            "k": torch.ones(self.size, device="cuda"),
            "scale": torch.ones(dim, device="cuda"),
            "shift": torch.zeros(dim, device="cuda"),
            "topics": make(topics, dim) / dim ** 0.5,
        }
        self.momentum = {name: torch.zeros_like(self.weights[name]) for name in ("qkv", "out")}
        self.frequencies = 1000.0 ** (-torch.arange(0, self.size, 2, device="cuda", dtype=torch.float32) / self.size)

    def encode(self, text):
        """The vectors of texts, and what their gradients need."""
        w, h, g = self.weights, self.heads, self.kv_heads
        tokens, offsets, positions = text
        x = w["words"][tokens]
        qkv = (x @ w["qkv"]).view(len(tokens), h + 2 * g, self.size)
        q, k, v = qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:]
        at = (q, k, w["q"], w["k"], positions, self.frequencies)
        a, b = training.qk_norm_rotary(*at)
        o, lse = training.attention(a, b, v, offsets)
        last = offsets[1:] - 1
        z = x[last] + o.flatten(1)[last] @ w["out"]
        y, mean, rstd = training.layer_norm(z, w["scale"], w["shift"])
        return y, (x, at, a, b, v, o, lse, last, z, mean, rstd)

    def gradients(self, text, topic):
        """The mean loss of texts of known topics, and the gradients of all weights."""
        w, h, g = self.weights, self.heads, self.kv_heads
        tokens, offsets, _ = text
        y, (x, at, a, b, v, o, lse, last, z, mean, rstd) = self.encode(text)
        each = torch.full((len(topic),), 1.0 / len(topic), device="cuda")
        loss, _, dy, dtopics = training.softmax_xent_grad(y, w["topics"], topic, each)
        dz, dscale, dshift = training.layer_norm_backward(dy, z, w["scale"], mean, rstd)
        do = torch.zeros_like(o)
        do[last] = (dz @ w["out"].t()).view(-1, h, self.size)
        da, db, dv = training.attention_backward(do, a, b, v, o, lse, offsets)
        dq, dk, dqw, dkw = training.qk_norm_rotary_backward(da, db, *at)
        dqkv = torch.cat((dq, dk, dv), 1).flatten(1)
        dx = dqkv @ w["qkv"].t()
        dx[last] += dz
        found = {
            "words": torch.zeros_like(w["words"]).index_add_(0, tokens, dx),
            "qkv": x.t() @ dqkv,
            "out": o.flatten(1)[last].t() @ dz,
            "q": dqw, "k": dkw, "scale": dscale, "shift": dshift, "topics": dtopics,
        }
        return loss.mean(), found

    def step(self, text, topic, rate=0.02, table_rate=20.0, beta=0.9, limit=0.5):
        """One step; the mean loss and the gradients' norm."""
        loss, found = self.gradients(text, topic)
        norm = training.clip_gradients(found.values(), limit)
        for name, d in found.items():
            if name in self.momentum:
                self.momentum[name].mul_(beta).add_(d)
                self.weights[name] -= rate * training.orthogonalize(self.momentum[name])
            else:
                self.weights[name] -= (table_rate if name in ("words", "topics") else rate) * d
        return loss, norm


def texts(count, topics, words, gen, longest=40):
    """Texts of 1 to `longest` words, mostly of those that their topic is about; their topics."""
    topic = torch.randint(0, topics, (count,), device="cuda", generator=gen)
    lengths = torch.randint(1, longest + 1, (count,), device="cuda", generator=gen)
    offsets = torch.zeros(count + 1, device="cuda", dtype=torch.int64)
    offsets[1:] = lengths.cumsum(0)
    n = int(offsets[-1])
    of = torch.repeat_interleave(torch.arange(count, device="cuda"), lengths)
    about = (topic[of] * 7919 + torch.randint(0, 8, (n,), device="cuda", generator=gen) * 104729) % words
    any_word = torch.randint(0, words, (n,), device="cuda", generator=gen)
    tokens = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.6, about, any_word)
    return (tokens, offsets, torch.arange(n, device="cuda") - offsets[of]), topic


def precision(encoder, text, topic, k=5):
    """Share of a text's k nearest others, by inner product, that are of its topic."""
    y = encoder.encode(text)[0].cpu().numpy()
    ids, _, _ = vh.CudaKnnEngine(y, metric=vh.DistanceMetric.DotProduct).search_batch_arrays(y, k + 1)
    near = torch.from_numpy(ids.astype("int64"))
    of, others = topic.cpu(), near != torch.arange(len(y))[:, None]
    return float(((of[near] == of[:, None]) & others).sum() / others.sum())


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--topics", type=int, default=200)
    p.add_argument("--words", type=int, default=5000)
    p.add_argument("--batch", type=int, default=512)
    p.add_argument("--steps", type=int, default=80)
    a = p.parse_args(argv)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    encoder = TextEncoder(a.words, a.topics)
    held = texts(2000, a.topics, a.words, gen)
    before = precision(encoder, *held)
    for step in range(a.steps):
        loss, norm = encoder.step(*texts(a.batch, a.topics, a.words, gen))
        if step % 20 == 0 or step + 1 == a.steps:
            print(f"step {step:4d}  loss {float(loss):.3f}  norm {float(norm):.3f}", flush=True)
    after = precision(encoder, *held)
    print(f"of the 5 nearest texts of {len(held[1])}, of the same topic: {before:.3f} before, {after:.3f} after")
    return before, after


if __name__ == "__main__":
    main()
