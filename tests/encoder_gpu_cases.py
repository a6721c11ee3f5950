"""Attention, head norms with rotation and gradient clipping (attention_forward.hip, attention_backward.hip,
head_norm.hip, clip.hip) against their definitions in 64 bits.

Tolerances are bounds of the arithmetic, made from the case's own values: u is half a unit of a type (a rounding
to it is off by u of the value at most), e = 2^-24 that of a 32-bit operation; a sum of n terms of absolute sum s is
held to n e s.

test_encoder_gpu.py runs this file in a process of its own, where torch is imported before the library: torch
brings a HIP runtime, and the other GPU tests want a process with the library's own."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


@pytest.fixture(scope="module")
def tr():
    import vector_hip

    assert vector_hip.CudaDeviceContext.device_count() >= 1
    from vector_hip import training

    return training


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(seed, *shape):
    return torch.randn(*shape, device="cuda", generator=gen(seed))


def within(got, want, tol):
    """Every value within tol; where want is not finite, the same."""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    off = torch.where(fine, (got - want).abs() - tol, torch.full_like(want, -1.0))
    assert off.numel() == 0 or float(off.max()) <= 0, f"over the tolerance by {float(off.max()):.3g}"


# ---- attention --------------------------------------------------------------------------------------

def ends(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def bounds(lengths):
    return torch.tensor(ends(lengths), device="cuda", dtype=torch.int64)


def attention_case(lq, lk, heads, kv, dim, dtype, seed=0, tail=0, size=1.0):
    """Inputs with `tail` rows of no sequence."""
    tq, tk = sum(lq) + tail, sum(lk) + tail
    t = TYPES[dtype]
    q, k, v, do = ((size * normal(seed + i, n, h, dim)).to(t) for i, (n, h) in enumerate([(tq, heads), (tk, kv), (tk, kv), (tq, heads)]))
    return q, k, v, do


def attention_reference(q, k, v, lq, lk, causal, scale, do=None):
    """out, lse, their tolerances, and with do the gradients of q, k, v with theirs, all in 64 bits.

    A score of a = scale |q|.|k| is off by (dim + 8) e a: its sum's chain, the scale, the largest one taken off.
    lse is off by the scores' mean of that, by the row's sum (m e), by exp's and log's own 8 e and by 4 e |lse|; a
    weight by its score and that, and by u where it is rounded to be multiplied.  The backward pass makes p from the
    rounded lse: twice lse's error.  ds = p (dp - delta) has the errors of p, of dp and of delta, which takes the
    rounded out, and is rounded to be multiplied; in float16 it loses 2^-39 of its row's or key's largest one, and p 2^-39.
    Sums of m keys, or of all rows of a key, have that many e more."""
    t = q.dtype
    u, tiny, wide = UNIT[t], TINY[t], t == torch.float32
    up = 0.0 if wide else u  # of p and ds as operands
    lost = 2.0 ** -39 if t == torch.float16 else 0.0
    heads, dim = q.shape[1], q.shape[2]
    per = heads // k.shape[1]
    z = lambda x: torch.zeros(x.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    r = {"out": z(q), "lse": torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")}
    tol = {"out": z(q) + tiny, "lse": z(r["lse"])}
    if do is not None:
        for n, x in (("dq", q), ("dk", k), ("dv", v)):
            r[n], tol[n] = z(x), z(x) + tiny
    qb = kb = 0
    for n, m in zip(lq, lk):
        rows, keys = slice(qb, qb + n), slice(kb, kb + m)
        for h in range(heads if n and m else 0):
            Q, K, V = q[rows, h].double(), k[keys, h // per].double(), v[keys, h // per].double()
            seen = torch.ones(n, m, device="cuda", dtype=torch.bool)
            if causal:
                seen = seen.tril(m - n)
            s = (Q @ K.t() * scale).masked_fill(~seen, -math.inf)
            off = ((dim + 8) * E * abs(scale) * (Q.abs() @ K.abs().t())).masked_fill(~seen, 0.0)
            lse = torch.logsumexp(s, 1)
            safe = torch.where(seen.any(1), lse, torch.zeros_like(lse))
            p = torch.where(seen, torch.exp(s - safe[:, None]), 0.0)
            o, osize = p @ V, p @ V.abs()
            elses = (p * off).sum(1) + (m + 8) * E + 4 * E * safe.abs()
            rel = off + elses[:, None]
            r["out"][rows, h], r["lse"][rows, h] = o, lse
            tol["out"][rows, h] += (p * (rel + up)) @ V.abs() + (m + 8) * E * osize + u * o.abs() + lost * V.abs().sum(0)
            tol["lse"][rows, h] = torch.where(seen.any(1), elses, torch.zeros_like(elses))
            if do is None:
                continue
            G, rel = do[rows, h].double(), off + 2 * elses[:, None]
            dp, delta = G @ V.t(), (G * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            edp = (dim + 4) * E * (G.abs() @ V.abs().t() + (G.abs() * osize).sum(1, keepdim=True))
            edelta = (G.abs() * tol["out"][rows, h]).sum(1, keepdim=True)
            eds = p * (edp + edelta) + (rel + up + 4 * E) * ds.abs()
            top = lambda x, d: lost * x.abs().amax(d, keepdim=True)  # noqa: E731
            a = abs(scale)
            r["dq"][rows, h] = scale * ds @ K
            tol["dq"][rows, h] += a * (eds + top(ds, 1) + (m + 8) * E * ds.abs()) @ K.abs() + u * r["dq"][rows, h].abs()
            more = (per * n + 8) * E
            r["dk"][keys, h // per] += scale * ds.t() @ Q
            tol["dk"][keys, h // per] += a * (eds + top(ds, 0) + more * ds.abs()).t() @ Q.abs()
            r["dv"][keys, h // per] += p.t() @ G
            tol["dv"][keys, h // per] += (p * (rel + up) + lost + more * p).t() @ G.abs()
        for x in ("dk", "dv") if do is not None else ():
            tol[x][keys] += u * r[x][keys].abs()
        qb, kb = qb + n, kb + m
    return r, tol


# lengths of queries and keys, heads, key heads, dim
ATTENTION = [
    ([1], [1], 1, 1, 1), ([19], [19], 12, 12, 64), ([3, 0, 5, 1], [3, 0, 5, 1], 2, 1, 32), ([64, 65, 63], [64, 65, 63], 4, 2, 72),
    ([200, 31], [200, 31], 3, 1, 100), ([129], [129], 8, 2, 128), ([300, 17], [300, 17], 6, 2, 33), ([1, 1, 1], [70, 1, 333], 8, 2, 128),
    ([5, 9, 4], [4, 700, 0], 4, 4, 64), ([40, 7], [90, 130], 5, 1, 96), ([513], [513], 2, 2, 31), ([2, 3] * 70, [2, 3] * 70, 1, 1, 16),
    ([1, 2], [5000, 3000], 4, 1, 64), ([3], [2100], 2, 2, 80),
]


@pytest.mark.parametrize("lq,lk,heads,kv,dim", ATTENTION)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention(tr, lq, lk, heads, kv, dim, causal, dtype):
    print("attention", lq[:4], lk[:4], heads, kv, dim, causal, dtype, flush=True)
    q, k, v, _ = attention_case(lq, lk, heads, kv, dim, dtype, tail=3)
    scale = 1 / math.sqrt(dim)
    out, lse = tr.attention(q, k, v, bounds(lq), None if lq == lk else bounds(lk), causal=causal)
    want, tol = attention_reference(q, k, v, lq, lk, causal, scale)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    within(out, want["out"], tol["out"])
    within(lse, want["lse"], tol["lse"])


@pytest.mark.parametrize("lq,lk,heads,kv,dim", ATTENTION)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_backward(tr, lq, lk, heads, kv, dim, causal, dtype):
    print("attention_backward", lq[:4], lk[:4], heads, kv, dim, causal, dtype, flush=True)
    q, k, v, do = attention_case(lq, lk, heads, kv, dim, dtype, tail=3)
    scale = 1 / math.sqrt(dim)
    at, kat = bounds(lq), None if lq == lk else bounds(lk)
    out, lse = tr.attention(q, k, v, at, kat, causal=causal)
    want, tol = attention_reference(q, k, v, lq, lk, causal, scale, do)
    for name, got in zip(("dq", "dk", "dv"), tr.attention_backward(do, q, k, v, out, lse, at, kat, causal=causal)):
        assert got.dtype == q.dtype
        within(got, want[name], tol[name])
