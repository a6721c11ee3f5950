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


# ---- what else a call may be given -------------------------------------------------------------------

def attention_both(tr, q, k, v, do, at, kat, causal, scale=None):
    out, lse = tr.attention(q, k, v, at, kat, causal=causal, scale=scale)
    return (out, lse) + tuple(tr.attention_backward(do, q, k, v, out, lse, at, kat, causal=causal, scale=scale))


def check_attention(got, want, tol, names=("out", "lse", "dq", "dk", "dv")):
    for name, x in zip(names, got):
        within(x, want[name], tol[name])


@pytest.mark.parametrize("layout", ["heads first", "padded", "odd addresses", "one buffer"])
@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("bf16", 64), ("f16", 40), ("bf16", 33)])
def test_attention_layouts(tr, layout, dtype, dim):
    """The same values in other places, bit by bit."""
    lq, heads, kv = [70, 3, 130], 6, 2
    q, k, v, do = attention_case(lq, lq, heads, kv, dim, dtype)

    def place(x):
        n, h, d = x.shape
        if layout == "heads first":
            return x.transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "padded":
            y = torch.full((n, h + 1, d + 24), math.nan, device="cuda", dtype=x.dtype)[:, :h, :d]
        elif layout == "odd addresses":
            y = torch.full((n * h * (d + 1) + 1,), math.nan, device="cuda", dtype=x.dtype)[1:].view(n, h, d + 1)[..., :d]
        else:
            y = torch.full((n, 3 * h, d), math.nan, device="cuda", dtype=x.dtype)[:, h:2 * h]
        y.copy_(x)
        return y

    at = bounds(lq)
    want = attention_both(tr, q, k, v, do, at, None, True)
    got = attention_both(tr, place(q), place(k), place(v), place(do), at, None, True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_attention_scales(tr, dtype, scale):
    lq, heads, kv, dim = [40, 100], 4, 2, 48
    q, k, v, do = attention_case(lq, lq, heads, kv, dim, dtype)
    want, tol = attention_reference(q, k, v, lq, lq, True, scale, do)
    check_attention(attention_both(tr, q, k, v, do, bounds(lq), None, True, scale), want, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1e-3, 8.0])
def test_attention_flat_and_peaked_rows(tr, dtype, size):
    lq, heads, kv, dim = [300], 2, 1, 64
    q, k, v, do = attention_case(lq, lq, heads, kv, dim, dtype, size=size)
    scale = 1 / math.sqrt(dim)
    want, tol = attention_reference(q, k, v, lq, lq, False, scale, do)
    check_attention(attention_both(tr, q, k, v, do, bounds(lq), None, False), want, tol)


@pytest.mark.parametrize("power", [-14, -20, 12])
def test_attention_gradients_of_any_size_in_float16(tr, power):
    """ds has powers of two of its own: gradients of small out gradients keep their bits."""
    lq, heads, kv, dim = [90, 260], 2, 1, 64
    q, k, v, do = attention_case(lq, lq, heads, kv, dim, "f16")
    do = (do.float() * 2.0 ** power).half()
    v = (v.float() * 2.0 ** -4).half()
    scale = 1 / math.sqrt(dim)
    want, tol = attention_reference(q, k, v, lq, lq, True, scale, do)
    check_attention(attention_both(tr, q, k, v, do, bounds(lq), None, True), want, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_sequences_do_not_meet(tr, dtype, causal):
    """What other sequences hold, and rows of none, changes nothing: not a bit."""
    lq, heads, kv, dim = [50, 33, 77], 4, 2, 64
    q, k, v, do = attention_case(lq, lq, heads, kv, dim, dtype, tail=20)
    at = bounds(lq)
    want = attention_both(tr, q, k, v, do, at, None, causal)
    for bad in (math.nan, math.inf):
        x = [y.clone() for y in (q, k, v, do)]
        for y in x:
            y[50:83] = bad
            y[160:] = bad
        got = attention_both(tr, *x, at, None, causal)
        for a, b in zip(got, want):
            assert torch.equal(a[:50], b[:50]) and torch.equal(a[83:160], b[83:160])
            assert torch.equal(a[160:], torch.full_like(a[160:], -math.inf) if a.dim() == 2 else torch.zeros_like(a[160:]))


def test_offsets_that_skip_rows_or_fall(tr):
    """Rows before the first and behind the last sequence come out empty; offsets out of the arrays reach nothing."""
    q, k, v, do = attention_case([100], [100], 2, 1, 32, "bf16")
    at = torch.tensor([10, 40, 90], device="cuda")
    out, lse, dq, dk, dv = attention_both(tr, q, k, v, do, at, None, True)
    inner = attention_both(tr, *(x[10:90].clone() for x in (q, k, v, do)), at - 10, None, True)
    for a, b in zip((out, lse, dq, dk, dv), inner):
        assert torch.equal(a[10:90], b)
        assert torch.equal(a[:10], torch.full_like(a[:10], -math.inf) if a.dim() == 2 else torch.zeros_like(a[:10]))
    for wild in ([-5, 40, 1 << 40], [100, 0, 100], [50, 20, 10], [-(1 << 62), 7, 3]):
        attention_both(tr, q, k, v, do, torch.tensor(wild, device="cuda"), None, True)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_parts_of_the_keys_and_rows(tr, dtype):
    """Few rows against many keys, and many rows against few keys: sums over parts."""
    for lq, lk, heads, kv, causal in (([3, 1], [9000, 40], 8, 2, True), ([5000], [30], 2, 1, False), ([2, 700], [6000, 700], 4, 4, True)):
        print("parts", lq, lk, dtype, flush=True)
        q, k, v, do = attention_case(lq, lk, heads, kv, 64, dtype, tail=2)
        want, tol = attention_reference(q, k, v, lq, lk, causal, 0.125, do)
        check_attention(attention_both(tr, q, k, v, do, bounds(lq), bounds(lk), causal), want, tol)


def test_attention_gradient_against_differences(tr):
    """A step along a direction changes sum(do out) by what the gradients say."""
    lq, h = [30, 45], 1e-3
    q, k, v, do = attention_case(lq, lq, 4, 2, 32, "f32")
    at = bounds(lq)
    out, lse, dq, dk, dv = attention_both(tr, q, k, v, do, at, None, True)
    for x, g in ((q, dq), (k, dk), (v, dv)):
        u = normal(50, *x.shape)
        said = float((g.double() * u.double()).sum())
        found = 0.0
        for s in (1, -1):
            moved = [y if y is not x else (x + s * h * u) for y in (q, k, v)]
            want, _ = attention_reference(*moved, lq, lq, True, 1 / math.sqrt(32))
            found += s * float((want["out"] * do.double()).sum()) / (2 * h)
        # third derivatives: h^2 of the size of the sum's terms; 32-bit rounding of moved inputs over 2 h
        size = float((g.double().abs() * u.double().abs()).sum()) + float((do.double().abs() * out.double().abs()).sum())
        assert abs(said - found) <= (10 * h * h + 64 * E / h) * size


def test_keys_past_32_bits(tr):
    """A cache of more than 4 GiB; the sequence at its end."""
    tokens, kv, dim, n = 4_500_000, 8, 64, 700
    k = torch.zeros(tokens, kv, dim, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    q, ks, vs, do = attention_case([n], [n], 16, kv, dim, "bf16")
    k[-n:], v[-n:] = ks, vs
    at, kat = bounds([n]), torch.tensor([tokens - n, tokens], device="cuda")
    want = attention_both(tr, q, ks, vs, do, at, None, True)
    got = attention_both(tr, q, k, v, do, at, kat, True)
    ref, tol = attention_reference(q, ks, vs, [n], [n], True, 0.125, do)
    # both are within tol of the same value (a larger cache is read in other parts), so within 2 tol of each other
    within(got[0], want[0], 2 * tol["out"])
    check_attention((got[0], got[1], got[2], got[3][-n:], got[4][-n:]), ref, tol)
    assert not got[3][:-n].any() and not got[4][:-n].any()


def test_everything_is_repeatable(tr):
    lq = [513, 20, 77]
    q, k, v, do = attention_case(lq, lq, 6, 2, 64, "bf16")
    first = attention_both(tr, q, k, v, do, bounds(lq), None, True)
    x, y, w, pos, freq = head_norm_case(3000, 4, 2, 64, 64, 0, "bf16", "f32")
    heads = tr.qk_norm_rotary_backward(x.contiguous(), y.contiguous(), x, y, w[0], w[1], pos, freq)
    arrays = clip_arrays([3_000_001, 77, (33, 65)], ["f32", "bf16"])
    norm = tr.gradient_norm(arrays)
    for _ in range(5):
        for a, b in zip(first, attention_both(tr, q, k, v, do, bounds(lq), None, True)):
            assert torch.equal(a, b)
        for a, b in zip(heads, tr.qk_norm_rotary_backward(x.contiguous(), y.contiguous(), x, y, w[0], w[1], pos, freq)):
            assert torch.equal(a, b)
        assert torch.equal(norm, tr.gradient_norm(arrays))


# ---- head norms and clipping at their edges ----------------------------------------------------------

def test_head_norm_without_weights_and_far_positions(tr):
    q, k, _, _, _ = head_norm_case(50, 3, 1, 64, 64, 0, "f32", "f32")
    freq = torch.ones(32, device="cuda")
    pos = torch.tensor([0, 1, -1, 10**6, -10**9, 2**40, 2**52], device="cuda").repeat(8)[:50]
    got = tr.qk_norm_rotary(q, k, None, None, pos, freq)
    angle = pos.double()[:, None] * freq.double()
    for x, y in zip((q, k), got):
        want, tol = head_norm_reference(x, None, angle, False, 1e-6)
        # 2^52 radians: the reference's own reduction and this one's are exact to 2^52 2^-107
        within(y, want, tol + UNIT[y.dtype] * want.abs())
    dq, dk, dqw, dkw = tr.qk_norm_rotary_backward(got[0], got[1], q, k, None, None, pos, freq)
    assert dqw is None and dkw is None
    # the gradient of half the squared norm of rows whose norm is fixed: only eps moves it
    assert float(dq.abs().max()) <= 1e-4 and float(dk.abs().max()) <= 1e-4


def test_head_norm_rows_of_zeros_and_one_bad_row(tr):
    q, k, w, pos, freq = head_norm_case(20, 2, 2, 48, 32, 0, "bf16", "f32")
    q, k = q.clone(), k.clone()
    want = tr.qk_norm_rotary(q, k, w[0], w[1], pos, freq)
    q[3], q[5], k[7] = 0, math.nan, math.inf
    got = tr.qk_norm_rotary(q, k, w[0], w[1], pos, freq)
    assert not got[0][3].any() and torch.isnan(got[0][5]).all() and torch.isnan(got[1][7]).all()
    keep = torch.ones(20, dtype=torch.bool, device="cuda")
    keep[[3, 5]] = False
    assert torch.equal(got[0][keep], want[0][keep])
    keep[:], keep[7] = True, False
    assert torch.equal(got[1][keep], want[1][keep])


def test_head_norm_gradient_against_differences(tr):
    q, k, w, pos, freq = head_norm_case(9, 3, 2, 40, 24, 0, "f32", "f32")
    dq, dk = normal(8, *q.shape), normal(9, *k.shape)
    got = tr.qk_norm_rotary_backward(dq, dk, q, k, w[0], w[1], pos, freq, eps=1e-3)
    angle, h = pos.double()[:, None] * freq.double(), 1e-4
    for x, wt, g, dx, dw in zip((q, k), w, (dq, dk), got[:2], got[2:]):
        u, uw = normal(20, *x.shape).double(), normal(21, *wt.shape).double()
        f = lambda s: float((head_norm_reference(x.double() + s * h * u, wt.double() + s * h * uw, angle, False, 1e-3)[0] * g.double()).sum())  # noqa: E731,B023
        said = float((dx.double() * u).sum() + (dw.double() * uw).sum())
        size = float((dx.double().abs() * u.abs()).sum() + (dw.double().abs() * uw.abs()).sum())
        assert abs(said - (f(1) - f(-1)) / (2 * h)) <= (1e3 * h * h + 64 * E) * (size + float(g.abs().sum()))


@pytest.mark.parametrize("dtype,value", [("f32", 3e38), ("f32", 1e-40), ("f32", 1e25), ("bf16", 1e38), ("bf16", 1e-38), ("f16", 65504.0), ("f16", 6e-8)])
def test_clip_values_of_any_size(tr, dtype, value):
    a = torch.full((1000,), value, device="cuda").to(TYPES[dtype])
    norm, c = clip_reference([a], 1.0, 0.0)
    got = tr.gradient_norm([a])
    if float(norm) < 3.4e38:
        within(got, norm, 2 * E * norm + 2.0 ** -149)
    else:
        assert math.isinf(float(got))
    b = a.clone()
    tr.clip_gradients([b], 1.0, eps=0.0)
    want = a.double() * float(c)
    # c itself is rounded to 32 bits, where it may have lost bits below 2^-126
    within(b, want, (2 * E + UNIT[b.dtype] + 2.0 ** -149 / max(float(c), 1e-300)) * want.abs() + TINY[b.dtype] + (2.0 ** -126 if dtype == "f32" else 0))


def test_clip_norms_that_are_not_finite(tr):
    for bad in (math.inf, -math.inf, math.nan):
        a, b = torch.ones(3000, device="cuda"), torch.ones(5, device="cuda", dtype=torch.bfloat16)
        a[7] = bad
        norm = tr.clip_gradients([a, b], 1.0)
        if math.isnan(bad):
            assert math.isnan(float(norm)) and torch.isnan(a).all() and torch.isnan(b).all()
        else:
            assert math.isinf(float(norm)) and torch.isnan(a[7]) and not b.any() and int((a == 0).sum()) == 2999


def test_clip_dense_arrays_in_other_orders(tr):
    a = normal(1, 40, 50).t()
    o = torch.empty(40, 50, device="cuda").t()
    want = a.double() * min(1.0, 1.0 / float(a.double().norm()))
    tr.clip_gradients([a, a[:0]], 1.0, out=[o, a[:0]], eps=0.0)
    within(o, want, 4 * E * want.abs())


# ---- streams, graphs, refusals ----------------------------------------------------------------------

def encoder_calls(tr, dtype="bf16"):
    """All operators as a step has them one after the other, as a function without arguments."""
    lq = [60, 133, 5]
    at = bounds(lq)
    q, k, v, do = attention_case(lq, lq, 4, 2, 64, dtype)
    _, _, w, pos, freq = head_norm_case(sum(lq), 4, 2, 64, 64, 0, dtype, dtype)
    few_q, few_k = bounds([1, 2]), bounds([5000, 100])
    fq, fk, fv, fdo = attention_case([1, 2], [5000, 100], 4, 2, 64, dtype)

    def run():
        a, b = tr.qk_norm_rotary(q, k, w[0], w[1], pos, freq)
        out, lse = tr.attention(a, b, v, at)
        da, db, dv = tr.attention_backward(do, a, b, v, out, lse, at)
        dq, dk, dqw, dkw = tr.qk_norm_rotary_backward(da, db, q, k, w[0], w[1], pos, freq)
        clipped = [torch.empty_like(x) for x in (dq, dk, dv, dqw, dkw)]
        norm = tr.clip_gradients([dq, dk, dv, dqw, dkw], 0.5, out=clipped)
        few = attention_both(tr, fq, fk, fv, fdo, few_q, few_k, True)
        return [out, lse, norm, *clipped, *few]

    return run


def test_calls_on_another_stream(tr):
    run = encoder_calls(tr)
    want = run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    other = run()  # at the same time
    torch.cuda.synchronize()
    for a, b, c in zip(got, want, other):
        assert torch.equal(a, b) and torch.equal(c, b)


def test_calls_in_graphs(tr):
    """Two captured graphs, replayed in turn and with eager work between."""
    runs = [encoder_calls(tr, "bf16"), encoder_calls(tr, "f16")]
    want = [run() for run in runs]
    graphs, got = [], []
    for run in runs:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(run())
        graphs.append(g)
    for _ in range(4):
        for g, outs, w, run in zip(graphs, got, want, runs):
            for x in outs:
                x.zero_()
            g.replay()
            eager = run()
            torch.cuda.synchronize()
            for a, b, c in zip(outs, w, eager):
                assert torch.equal(a, b) and torch.equal(c, b)


def test_refusals(tr):
    import vector_hip as vh

    q, k, v, do = attention_case([9], [9], 4, 2, 32, "bf16")
    at = bounds([9])
    out, lse = tr.attention(q, k, v, at)
    w, pos, freq = torch.ones(32, device="cuda", dtype=torch.bfloat16), torch.arange(9, device="cuda"), torch.ones(16, device="cuda")
    norm = lambda *a, **o: tr.qk_norm_rotary(*a, **o)  # noqa: E731
    big = torch.zeros(2, 1, 129, device="cuda")
    wrong = [
        lambda: tr.attention(q, k, v, at.int()), lambda: tr.attention(q, k, v, at.cpu()), lambda: tr.attention(q, k, v, at[:0]),
        lambda: tr.attention(q[0], k, v, at), lambda: tr.attention(q, k.float(), v, at), lambda: tr.attention(q, k, v[:, :1], at),
        lambda: tr.attention(q[:, :3], k, v, at), lambda: tr.attention(q, k[..., :16], v[..., :16], at), lambda: tr.attention(q, k[:5], v[:5], at),
        lambda: tr.attention(q, k, v, at, at[:1]), lambda: tr.attention(q, k, v, at, scale=math.inf), lambda: tr.attention(q, k, v, at, scale=math.nan),
        lambda: tr.attention(q.long(), k.long(), v.long(), at), lambda: tr.attention(big, big, big, bounds([2])),
        lambda: tr.attention(q[..., ::2], k[..., ::2], v[..., ::2], at), lambda: tr.attention(q, k[:1].expand(9, 2, 32), v, at),
        lambda: tr.attention(q.requires_grad_(), k, v, at), lambda: tr.attention(q.cpu(), k.cpu(), v.cpu(), at.cpu()),
        lambda: tr.attention_backward(do[:5], q, k, v, out, lse, at), lambda: tr.attention_backward(do, q, k, v, out[:, :2], lse, at),
        lambda: tr.attention_backward(do, q, k, v, out, lse.t(), at), lambda: tr.attention_backward(do, q, k, v, out, lse.double(), at),
        lambda: norm(q, k, w, None, pos, freq), lambda: norm(q, k, w, w.float(), pos, freq), lambda: norm(q, k, w.half(), w.half(), pos, freq),
        lambda: norm(q, k, w[:5], w[:5], pos, freq), lambda: norm(q, k, w, w, pos[:5], freq), lambda: norm(q, k, w, w, pos.int(), freq),
        lambda: norm(q, k, w, w, pos, freq.double()), lambda: norm(q, k, w, w, pos, torch.ones(17, device="cuda")), lambda: norm(q, k[:4], w, w, pos, freq),
        lambda: norm(q, k, w, w, pos, freq, eps=-1.0), lambda: norm(q, k.half(), w, w, pos, freq),
        lambda: norm(torch.zeros(9, 2, 257, device="cuda"), torch.zeros(9, 2, 257, device="cuda"), None, None, pos, freq),
        lambda: tr.qk_norm_rotary_backward(do[:4], k, q, k, w, w, pos, freq),
        lambda: tr.clip_gradients([], 1.0), lambda: tr.clip_gradients([q, q], 1.0), lambda: tr.clip_gradients([q.detach(), q.detach()[3:]], 1.0),
        lambda: tr.clip_gradients([do], -1.0), lambda: tr.clip_gradients([do], math.nan), lambda: tr.clip_gradients([do], 1.0, eps=-1.0),
        lambda: tr.clip_gradients([do[:, ::2]], 1.0), lambda: tr.clip_gradients([do, at], 1.0), lambda: tr.clip_gradients([do], 1.0, out=[]),
        lambda: tr.clip_gradients([do], 1.0, out=[do[:4]]), lambda: tr.clip_gradients([do, k], 1.0, out=[k, do.float()]),
        lambda: tr.clip_gradients([do, k], 1.0, out=[k[:0].new_empty(do.shape), do.view(-1)[:k.numel()].view(k.shape)]),
        lambda: tr.clip_gradients([do.cpu()], 1.0), lambda: tr.gradient_norm([do, do.cpu()]),
    ]
    for i, call in enumerate(wrong):
        with pytest.raises(vh.InvalidConfig):
            call()
            pytest.fail(f"call {i} was not refused")
        q = q.detach()
    with torch.no_grad():
        tr.attention(q.requires_grad_(), k, v, at)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (6, 2, 128), (3, 1, 40)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_counts_for_nothing(tr, dtype, heads, kv, dim, bad):
    """Causal: keys and values behind a row may hold anything; the row keeps its bits."""
    print("not seen", dtype, heads, kv, dim, bad, flush=True)
    lq, cut = [150, 300], 83
    q, k, v, _ = attention_case(lq, lq, heads, kv, dim, dtype)
    out, lse = tr.attention(q, k, v, bounds(lq))
    for which in ("kv", "k", "v"):
        x, y = k.clone(), v.clone()
        if "k" in which:
            x[cut:150] = bad
        if "v" in which:
            y[cut:150] = bad
        got, gl = tr.attention(q, x, y, bounds(lq))
        keep = torch.ones(450, dtype=torch.bool, device="cuda")
        keep[cut:150] = False
        assert torch.equal(got[keep], out[keep]) and torch.equal(gl[keep], lse[keep])
        assert which == "k" or not torch.isfinite(got[cut:150]).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_infinities_that_are_seen(tr, dtype):
    """An infinite value comes out in the rows that see it, in its column; both signs together are NaN."""
    n = 100
    q, k, v, do = attention_case([n], [n], 2, 2, 64, dtype)
    v[40, 0, 5], v[60, 1, 9], v[70, 1, 9] = math.inf, -math.inf, math.inf
    for causal in (True, False):
        out, _ = tr.attention(q, k, v, bounds([n]), causal=causal)
        want = torch.zeros(n, 2, 64, device="cuda")
        want[(40 if causal else 0):, 0, 5] = math.inf
        want[(60 if causal else 0):, 1, 9] = -math.inf
        want[(70 if causal else 0):, 1, 9] = math.nan
        bad = ~torch.isfinite(want)
        assert torch.equal(~torch.isfinite(out), bad)
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[torch.isinf(want)].float(), want[torch.isinf(want)])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(160, 1, 16), (128, 1, 64), (192, 2, 24), (7, 7, 128), (65, 13, 8)])
def test_groups_of_any_size(tr, dtype, heads, kv, dim):
    """Groups wider than a tile of rows, and of sizes that divide nothing."""
    print("groups", heads, kv, dim, dtype, flush=True)
    lq = [5, 0, 41, 1]
    q, k, v, do = attention_case(lq, lq, heads, kv, dim, dtype)
    for causal in (True, False):
        want, tol = attention_reference(q, k, v, lq, lq, causal, 1 / math.sqrt(dim), do)
        check_attention(attention_both(tr, q, k, v, do, bounds(lq), None, causal), want, tol)


def test_no_sequences_and_no_rows(tr):
    q, k, v, do = attention_case([6], [6], 4, 2, 32, "bf16")
    none = torch.zeros(1, device="cuda", dtype=torch.int64)
    out, lse, dq, dk, dv = attention_both(tr, q, k, v, do, none, None, True)
    assert not out.any() and torch.isinf(lse).all() and not dq.any() and not dk.any() and not dv.any()
    at, kat = bounds([0, 0]), bounds([4, 2])
    out, lse, dq, dk, dv = attention_both(tr, q[:0], k, v, do[:0], at, kat, False)
    assert out.shape == (0, 4, 32) and not dk.any() and not dv.any()
    out, lse, dq, dk, dv = attention_both(tr, q, k[:0], v[:0], do, kat, at, False)
    assert not out.any() and torch.isinf(lse).all() and not dq.any() and dk.shape == (0, 2, 32)
    out, lse, dq, dk, dv = attention_both(tr, q[:0], k[:0], v[:0], do[:0], none, None, True)
    assert dv.shape == (0, 2, 32)


def test_angles_that_are_none(tr):
    """A product of position and frequency past 2^52 has no angle: NaN in the pairs, and nowhere else."""
    q, k, _, _, _ = head_norm_case(3, 2, 1, 16, 8, 0, "f32", "f32")
    pos = torch.tensor([5, 2**53, 2**62], device="cuda")
    a, b = tr.qk_norm_rotary(q, k, None, None, pos, torch.tensor([1.0, 2.0, 1e3, 1e30], device="cuda"))
    for y in (a, b):
        bad = torch.isnan(y)
        assert not bad[..., 8:].any() and not bad[0, :, :3].any() and bad[0, :, 3].all() and bad[1:, :, :8].all()


# ---- the operators together --------------------------------------------------------------------------

def test_an_encoder_with_its_gradients(tr):
    """A step of examples/train_text_encoder.py against automatic differentiation of the same encoder in 64 bits."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_text_encoder.py")
    spec = importlib.util.spec_from_file_location("train_text_encoder", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    encoder = ex.TextEncoder(300, 20, seed=3)
    text, topic = ex.texts(40, 20, 300, gen(9))
    loss, found = encoder.gradients(text, topic)

    tokens, offsets, positions = text
    w = {name: x.double().requires_grad_() for name, x in encoder.weights.items()}
    h, g, d = encoder.heads, encoder.kv_heads, encoder.size
    x = w["words"][tokens]
    qkv = (x @ w["qkv"]).view(len(tokens), h + 2 * g, d)
    angle = positions.double()[:, None] * encoder.frequencies.double()
    z = []
    rows = [(int(b), int(e)) for b, e in zip(offsets, offsets[1:])]
    for b, e in rows:
        sides = []
        for part, weight in ((qkv[b:e, :h], w["q"]), (qkv[b:e, h:h + g], w["k"])):
            n = part / torch.sqrt((part * part).mean(2, keepdim=True) + 1e-6) * weight
            c, s = torch.cos(angle[b:e])[:, None], torch.sin(angle[b:e])[:, None]
            lo, hi = n[..., :d // 2], n[..., d // 2:]
            sides.append(torch.cat((lo * c - hi * s, lo * s + hi * c), 2))
        q, k = sides
        k, v = (y.repeat_interleave(h // g, 1) for y in (k, qkv[b:e, h + g:]))
        p = torch.softmax((k * q[-1]).sum(2) / d ** 0.5, 0)  # the last word sees all
        z.append(x[e - 1] + (p[..., None] * v).sum(0).flatten() @ w["out"])
    z = torch.stack(z)
    y = torch.nn.functional.layer_norm(z, (z.shape[1],), w["scale"], w["shift"], 1e-5)
    want = torch.nn.functional.cross_entropy(y @ w["topics"].t(), topic)
    assert abs(float(loss) - float(want.detach())) <= 1e-5 * float(want.detach())
    # a chain of ten operators in 32 bits, sums of up to 2000 terms: 2000 e of the gradient's largest values
    for name, got in zip(found, torch.autograd.grad(want, [w[n] for n in found])):
        within(found[name], got, 2000 * E * (got.abs() + got.abs().max()))
    before = [x.clone() for x in found.values()]
    norm, _ = clip_reference(before, 0.5, 1e-6)
    within(encoder.step(text, topic)[1], norm, 4 * E * norm)
