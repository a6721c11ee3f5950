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


# ---- head norms with rotation -----------------------------------------------------------------------

def turn(x, angle, interleaved, back=False):
    """Rows [tokens, heads, dim] with their first pairs turned, in 64 bits."""
    rot = 2 * angle.shape[1]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None] * (-1 if back else 1)
    y = x.clone()
    ya, yb = a * c - b * s, a * s + b * c
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = ya, yb
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = ya, yb
    return y


def both_of_a_pair(x, pairs, interleaved):
    """For each column what its pair holds together."""
    rot = 2 * pairs
    y = x.clone()
    for a, b in ([(slice(0, rot, 2), slice(1, rot, 2))] if interleaved else [(slice(0, pairs), slice(pairs, rot))]):
        y[..., a] = y[..., b] = x[..., a] + x[..., b]
    return y


def head_norm_reference(x, w, angle, interleaved, eps, dy=None):
    """y or (dx, dw) in 64 bits with bounds: the sum of dim squares and the scale are off by (dim / 2 + 6) e, sine and
    cosine by 4 e of a whole, products and their sum by 4 e more; dx and dw likewise by their terms' sizes."""
    dim, pairs = x.shape[2], angle.shape[1]
    x, w = x.double(), torch.ones(dim, device="cuda", dtype=torch.float64) if w is None else w.double()
    r = 1 / torch.sqrt((x * x).mean(2, keepdim=True) + eps)
    rel = (dim / 2 + 6) * E
    if dy is None:
        n = x * r * w
        return turn(n, angle, interleaved), (rel + 8 * E) * both_of_a_pair(n.abs(), pairs, interleaved)
    dn = turn(dy.double(), angle, interleaved, back=True)
    size = both_of_a_pair(dy.double().abs(), pairs, interleaved)
    xh, u = x * r, dn * w
    usize = size * w.abs()
    m = (u * xh).mean(2, keepdim=True)
    msize = (usize * xh.abs()).mean(2, keepdim=True)
    dx = r * (u - xh * m)
    tol = r * (rel + 16 * E + dim * E) * (usize + xh.abs() * msize)
    chain = x.shape[0] * x.shape[1]
    return dx, tol, (dn * xh).sum((0, 1)), (chain * E + rel + 16 * E) * (size * xh.abs()).sum((0, 1))


# tokens, heads, key heads, dim, rotated columns, neighbouring pairs, padding between rows
HEAD_NORMS = [
    (1, 12, 12, 64, 64, False, 0), (5, 32, 8, 128, 128, False, 8), (17, 4, 2, 80, 40, True, 0), (9, 3, 1, 33, 32, False, 1),
    (3, 2, 2, 256, 64, False, 0), (2, 1, 1, 256, 256, True, 0), (130, 6, 2, 72, 72, True, 0), (40, 5, 5, 1, 0, False, 0),
    (7, 2, 1, 7, 6, False, 0), (300, 2, 2, 20, 6, True, 3), (3000, 3, 1, 96, 96, False, 0), (0, 4, 2, 64, 64, False, 0),
    (4, 4, 2, 64, 0, False, 0), (9000, 1, 1, 16, 16, True, 0), (2, 3, 0, 64, 64, False, 0), (3, 2, 1, 253, 150, False, 5), (3, 1, 2, 256, 2, True, 0),
]


def head_norm_case(tokens, heads, kv, dim, rot, pad, dtype, params, far=40_000):
    t = TYPES[dtype]
    x = (2 * normal(1, tokens, heads + kv, dim + pad)).to(t)[..., :dim]
    w = [(1 + 0.3 * normal(2 + i, dim)).to(TYPES[params]) for i in range(2)]
    pos = torch.randint(-far, far, (tokens,), device="cuda", generator=gen(5))
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float32) / max(rot, 1))
    return x[:, :heads], x[:, heads:], w, pos, freq


@pytest.mark.parametrize("tokens,heads,kv,dim,rot,near,pad", HEAD_NORMS)
@pytest.mark.parametrize("dtype,params", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
def test_head_norm(tr, tokens, heads, kv, dim, rot, near, pad, dtype, params):
    print("qk_norm_rotary", tokens, heads, kv, dim, rot, near, pad, dtype, params, flush=True)
    q, k, w, pos, freq = head_norm_case(tokens, heads, kv, dim, rot, pad, dtype, params)
    got = tr.qk_norm_rotary(q, k, w[0], w[1], pos, freq, eps=1e-5, interleaved=near)
    angle = pos.double()[:, None] * freq.double()
    u, tiny = UNIT[q.dtype], TINY[q.dtype]
    for x, y, wt in zip((q, k), got, w):
        want, tol = head_norm_reference(x, wt, angle, near, 1e-5)
        assert y.dtype == x.dtype and y.shape == x.shape
        within(y, want, tol + u * want.abs() + tiny)


@pytest.mark.parametrize("tokens,heads,kv,dim,rot,near,pad", HEAD_NORMS)
@pytest.mark.parametrize("dtype,params", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
def test_head_norm_backward(tr, tokens, heads, kv, dim, rot, near, pad, dtype, params):
    print("qk_norm_rotary_backward", tokens, heads, kv, dim, rot, near, pad, dtype, params, flush=True)
    q, k, w, pos, freq = head_norm_case(tokens, heads, kv, dim, rot, pad, dtype, params)
    dq, dk = normal(8, *q.shape).to(q.dtype), normal(9, *k.shape).to(q.dtype)
    got = tr.qk_norm_rotary_backward(dq, dk, q, k, w[0], w[1], pos, freq, eps=1e-5, interleaved=near)
    angle = pos.double()[:, None] * freq.double()
    for x, g, wt, dx, dw in zip((q, k), (dq, dk), w, got[:2], got[2:]):
        want, tol, wantw, tolw = head_norm_reference(x, wt, angle, near, 1e-5, g)
        assert dx.dtype == x.dtype and dw.dtype == wt.dtype
        within(dx, want, tol + UNIT[x.dtype] * want.abs() + TINY[x.dtype])
        within(dw, wantw, tolw + UNIT[wt.dtype] * wantw.abs() + TINY[wt.dtype])


# ---- clipping ---------------------------------------------------------------------------------------

def clip_arrays(sizes, dtypes, scale=1.0):
    return [(scale * normal(i, *((n,) if isinstance(n, int) else n))).to(TYPES[dtypes[i % len(dtypes)]]) for i, n in enumerate(sizes)]


def clip_reference(arrays, max_norm, eps):
    total = sum(((a.double() ** 2).sum() for a in arrays), torch.zeros((), device="cuda", dtype=torch.float64))
    norm = total.sqrt()
    return norm, torch.clamp(max_norm / (norm + eps), max=1.0)


CLIPS = [[1], [3, 5], [2047, 2048, 2049, 1], [(96, 128), (128,), (128,), (2000, 128)], [0, 7, 0], [1] * 300, [17, 4096] * 130,
         [3_000_001], [8193, (33, 65), 100_003, 2], [0]]


@pytest.mark.parametrize("sizes", CLIPS)
@pytest.mark.parametrize("dtypes", [("f32",), ("f16",), ("bf16",), ("bf16", "f32", "f16")])
@pytest.mark.parametrize("out", [None, "f32", "bf16"])
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_clip(tr, sizes, dtypes, out, max_norm):
    print("clip", sizes[:4], len(sizes), dtypes, out, max_norm, flush=True)
    arrays = clip_arrays(sizes, dtypes)
    norm, c = clip_reference(arrays, max_norm, 1e-6)
    before = [a.clone() for a in arrays]
    outs = None if out is None else [torch.full(a.shape, math.nan, device="cuda", dtype=TYPES[out]) for a in arrays]
    within(tr.gradient_norm(arrays), norm, 2 * E * norm)
    got = tr.clip_gradients(arrays, max_norm, out=outs)
    assert got.dtype == torch.float32 and got.shape == ()
    within(got, norm, 2 * E * norm)
    for a, b, o in zip(arrays, before, arrays if outs is None else outs):
        if outs is not None:
            assert torch.equal(a, b)
        want = b.double() * c
        within(o, want, (2 * E + UNIT[o.dtype]) * want.abs() + TINY[o.dtype])
        if float(c) == 1.0 and o.dtype == b.dtype:
            assert torch.equal(o, b)
