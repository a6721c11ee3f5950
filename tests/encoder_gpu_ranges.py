"""Attention, head norms and clipping where values, sizes and layouts are at their limits.  Definitions and tolerances are those
of encoder_gpu_cases.py; what is new is derived where it stands.

test_encoder_ranges_gpu.py runs this file in a process of its own, where torch is imported before the library."""
import math

import pytest

torch = pytest.importorskip("torch")

from encoder_gpu_cases import (E, TINY, TYPES, UNIT, attention_both, attention_case, attention_reference, bounds, clip_arrays,  # noqa: E402,F401
                               gen, head_norm_case, head_norm_reference, normal, tr, within)

pytestmark = pytest.mark.gpu


def odd_address(x):
    """The same values one element off a vector's alignment."""
    n, h, d = x.shape
    y = torch.full((n * h * (d + 1) + 1,), math.nan, device=x.device, dtype=x.dtype)[1:].view(n, h, d + 1)[..., :d]
    y.copy_(x)
    return y


# ---- infinities that are seen ------------------------------------------------------------------------------

@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype,dim", [("f32", 36), ("f32", 72), ("f32", 64), ("f16", 40), ("f16", 80), ("bf16", 72), ("bf16", 104), ("bf16", 128)])
def test_keys_of_weight_zero_by_an_infinite_score(tr, dtype, dim, odd):
    """A key whose last column is -inf where queries are positive has score -inf: the rows come out as without it.  Its own
    gradients are 0, and the queries' are 0 * inf in that column alone."""
    print("infinite keys", dtype, dim, odd, flush=True)
    n, heads, kv = 150, 4, 2
    q, k, v, do = attention_case([n], [n], heads, kv, dim, dtype)
    q[..., -1] = q[..., -1].abs() + 0.5
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[[3, 40, 89, 149]] = False
    k[~keep, :, -1] = -math.inf
    want, tol = attention_reference(q, k[keep], v[keep], [n], [n - 4], False, 1 / math.sqrt(dim), do)
    if odd:
        q, k, v, do = (odd_address(x) for x in (q, k, v, do))
    out, lse, dq, dk, dv = attention_both(tr, q, k, v, do, bounds([n]), None, False)
    within(out, want["out"], tol["out"])
    within(lse, want["lse"], tol["lse"])
    within(dq[..., :-1], want["dq"][..., :-1], tol["dq"][..., :-1])
    within(dk[keep], want["dk"], tol["dk"])
    within(dv[keep], want["dv"], tol["dv"])
    assert not dk[~keep].any() and not dv[~keep].any()


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype,dim", [("f32", 36), ("f32", 72), ("f16", 40), ("bf16", 72), ("bf16", 104), ("bf16", 128)])
def test_rows_whose_scores_are_all_minus_infinity(tr, dtype, dim, odd):
    """Such a row counts as one that sees no key, and the keys' gradients come from the others (its own column times 0 aside)."""
    print("rows of infinite scores", dtype, dim, odd, flush=True)
    n, heads, kv = 150, 2, 2
    q, k, v, do = attention_case([n], [n], heads, kv, dim, dtype)
    k[..., -1] = k[..., -1].abs() + 0.5
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[[5, 70, 149]] = False
    q[~keep, :, -1] = -math.inf
    want, tol = attention_reference(q[keep], k, v, [n - 3], [n], False, 1 / math.sqrt(dim), do[keep])
    if odd:
        q, k, v, do = (odd_address(x) for x in (q, k, v, do))
    out, lse, dq, dk, dv = attention_both(tr, q, k, v, do, bounds([n]), None, False)
    for name, x in (("out", out), ("lse", lse), ("dq", dq)):
        within(x[keep], want[name], tol[name])
    assert not out[~keep].any() and not dq[~keep].any() and (lse[~keep] == -math.inf).all()
    within(dk[..., :-1], want["dk"][..., :-1], tol["dk"][..., :-1])
    within(dv, want["dv"], tol["dv"])


# ---- bits that do not depend on other rows -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (6, 2, 128), (3, 1, 40)])
@pytest.mark.parametrize("size", [8.0, 100.0, 1000.0])
def test_keys_that_are_not_seen_move_no_bit(tr, dtype, heads, kv, dim, size):
    """Causal: rows before keys of far larger scores keep their bits, though rows of the same tile see them."""
    print("larger keys", dtype, heads, kv, dim, size, flush=True)
    lq, cut = [150, 300], 83
    q, k, v, _ = attention_case(lq, lq, heads, kv, dim, dtype)
    out, lse = tr.attention(q, k, v, bounds(lq))
    k[cut:150] = (k[cut:150].float() * size).to(k.dtype)
    got, gl = tr.attention(q, k, v, bounds(lq))
    keep = torch.ones(450, dtype=torch.bool, device="cuda")
    keep[cut:150] = False
    assert torch.equal(got[keep], out[keep]) and torch.equal(gl[keep], lse[keep])
    assert not torch.equal(got[cut:150], out[cut:150])


# ---- head norms of rows of any size ------------------------------------------------------------------------

ROWS = [(40, 4, 2, 128, 128, False), (33, 3, 1, 80, 40, True), (70, 2, 2, 20, 12, False), (9, 1, 1, 256, 64, True)]


def rows_of_sizes(tokens, heads, kv, dim, rot, dtype, size):
    """Every second row `size` times as large."""
    q, k, w, pos, freq = head_norm_case(tokens, heads, kv, dim, rot, 0, "f32", "f32")
    q, k = (x.double() for x in (q, k))
    q[::2], k[1::2] = q[::2] * size, k[1::2] * size
    return q.float().to(TYPES[dtype]), k.float().to(TYPES[dtype]), w, pos, freq


@pytest.mark.parametrize("tokens,heads,kv,dim,rot,near", ROWS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size,eps", [(1e17, 1e-6), (3e18, 0.0), (1e19, 1e-6), (1e25, 1e-6), (2e37, 1e-6), (2e37, 1e30), (1e-18, 0.0), (1e-21, 0.0), (1e-18, 1e-36),
                                      (1e-30, 0.0), (1e-30, 1e-6), (1e-39, 0.0)])
def test_head_norm_of_rows_of_any_size(tr, tokens, heads, kv, dim, rot, near, dtype, size, eps):
    """Rows whose squares are past the range of 32 bits, beside ordinary ones."""
    print("rows of size", size, eps, tokens, heads, kv, dim, rot, near, dtype, flush=True)
    q, k, w, pos, freq = rows_of_sizes(tokens, heads, kv, dim, rot, dtype, size)
    angle = pos.double()[:, None] * freq.double()
    got = tr.qk_norm_rotary(q, k, w[0], w[1], pos, freq, eps=eps, interleaved=near)
    for x, y, wt in zip((q, k), got, w):
        want, tol = head_norm_reference(x, wt, angle, near, eps)
        within(y, want, tol + UNIT[y.dtype] * want.abs() + TINY[y.dtype])


@pytest.mark.parametrize("tokens,heads,kv,dim,rot,near", ROWS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size,eps,dsize", [(1e17, 1e-6, 1.0), (1e19, 1e-6, 1.0), (1e25, 1e-6, 1.0), (2e37, 1e-6, 1.0), (2e37, 1e30, 1.0), (1e-18, 0.0, 1.0),
                                            (1e-21, 0.0, 1.0), (1e-18, 1e-36, 1.0), (1e-30, 0.0, 1.0), (1e15, 1e-6, 1e28), (2e37, 1e-6, 1e30), (1e-12, 0.0, 1e-32)])
def test_head_norm_backward_of_rows_of_any_size(tr, tokens, heads, kv, dim, rot, near, dtype, size, eps, dsize):
    print("gradients of rows of size", size, eps, dsize, tokens, heads, kv, dim, rot, near, dtype, flush=True)
    q, k, w, pos, freq = rows_of_sizes(tokens, heads, kv, dim, rot, dtype, size)
    dq, dk = ((dsize * normal(8 + i, *x.shape).double()).float().to(x.dtype) for i, x in enumerate((q, k)))
    angle = pos.double()[:, None] * freq.double()
    got = tr.qk_norm_rotary_backward(dq, dk, q, k, w[0], w[1], pos, freq, eps=eps, interleaved=near)
    for x, g, wt, dx, dw in zip((q, k), (dq, dk), w, got[:2], got[2:]):
        want, tol, wantw, tolw = head_norm_reference(x, wt, angle, near, eps, g)
        within(dx, want, tol + UNIT[x.dtype] * want.abs() + TINY[x.dtype])
        within(dw, wantw, tolw + UNIT[wt.dtype] * wantw.abs() + TINY[wt.dtype])


# ---- clipping and graphs of automatic differentiation ------------------------------------------------------

def test_arrays_that_are_clipped_count_as_changed(tr):
    """A graph that saved an array raises once the array was clipped or written to, as after torch's own operations."""
    import vector_hip as vh

    w, g, o = torch.ones(50, device="cuda", requires_grad=True), 10 * normal(1, 50), normal(2, 50)
    for call, saved in ((lambda: tr.clip_gradients([g], 1.0), g), (lambda: tr.clip_gradients([g], 1.0, out=[o]), o),
                        (lambda: tr.clip_gradients([g[:20], g[20:]], 1.0), g)):
        loss = (w * saved).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    # what is only read stays valid, and so does what a refused call was given
    loss, want = (w * g).sum(), g.clone()
    tr.gradient_norm([g])
    tr.clip_gradients([g], 1.0, out=[o])
    with pytest.raises(vh.InvalidConfig):
        tr.clip_gradients([g], -1.0)
    loss.backward()
    assert torch.equal(w.grad, want)


def test_outputs_that_require_a_gradient_are_refused(tr):
    import vector_hip as vh

    g, leaf = normal(1, 50), torch.zeros(50, device="cuda", requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(vh.InvalidConfig):
            tr.clip_gradients([g], 1.0, out=[out])
        assert not out.any()
    with torch.no_grad():
        tr.clip_gradients([g], 1e6, out=[leaf])
    assert torch.equal(leaf.detach(), g)
    with torch.inference_mode():  # arrays without a version
        a, b = g + 1, g + 1
        tr.clip_gradients([a], 1e6, out=[b])
        tr.clip_gradients([a], 1e6)
        assert torch.equal(a, b)


# ---- more workgroups than one launch has -------------------------------------------------------------------

def test_attention_over_more_sequences_than_a_launch_has_workgroups(tr):
    """A launch has fewer than 2^32 threads: 2^24 workgroups of 256.  1.1 million sequences of 16 key heads take more, most of
    them empty here; those that are not come out as in a call of their own."""
    count, heads, dim = 1_100_000, 16, 16
    at = torch.zeros(count + 1, device="cuda", dtype=torch.int64)
    lengths = {0: 5, 400_000: 3, 700_001: 7, count - 1: 4}
    for s, n in lengths.items():
        at[s + 1:] += n
    n = sum(lengths.values())
    q, k, v, do = attention_case([n], [n], heads, heads, dim, "bf16")
    want = attention_both(tr, q, k, v, do, bounds(list(lengths.values())), None, True)
    got = attention_both(tr, q, k, v, do, at, None, True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_head_norms_of_more_tokens_than_a_launch_has(tr):
    """2 tokens are a workgroup's: 2^25 tokens are more than a launch has."""
    tokens, dim = (1 << 25) + 5, 2
    q = normal(1, tokens, 1, dim).half()
    k = q.new_empty(tokens, 0, dim)
    pos, freq = torch.arange(tokens, device="cuda"), torch.ones(1, device="cuda")
    got = tr.qk_norm_rotary(q, k, None, None, pos, freq)[0]
    for b, e in ((0, 1 << 24), (1 << 24, 1 << 25), ((1 << 25) - 1001, tokens)):
        part = tr.qk_norm_rotary(q[b:e], k[b:e], None, None, pos[b:e], freq)[0]
        assert torch.equal(got[b:e], part)


# ---- clipping: limits and norms whose quotient is none -----------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("out", [False, True])
def test_clip_limits_of_zero_and_infinity(tr, dtype, out):
    def clipped(values, max_norm, eps):
        arrays = [torch.tensor(x, device="cuda").to(TYPES[dtype]) for x in values]
        outs = [torch.full_like(a, 7.0) for a in arrays] if out else None
        norm = tr.clip_gradients(arrays, max_norm, out=outs, eps=eps)
        return float(norm), [a.tolist() for a in (outs or arrays)]

    nan, inf = math.nan, math.inf
    zeros, ordinary = [[0.0, 0.0, 0.0], [0.0]], [[3.0, 0.0], [4.0]]
    # zeros have norm 0, which a limit of 0 allows
    assert clipped(zeros, 0.0, 0.0) == (0.0, zeros)
    assert clipped(zeros, 0.0, 1e-6) == (0.0, zeros)
    assert clipped(ordinary, 0.0, 0.0) == (5.0, [[0.0, 0.0], [0.0]])
    assert clipped(ordinary, 5.0, 0.0) == (5.0, ordinary)
    assert clipped(ordinary, inf, 0.0) == (5.0, ordinary)
    # an infinite norm gives zeros, and NaN for the infinite values, whatever the limit
    for limit in (0.0, 1.0, inf):
        norm, ((a, b), (c,)) = clipped([[inf, 2.0], [3.0]], limit, 0.0)
        assert norm == inf and math.isnan(a) and b == 0.0 and c == 0.0
        norm, got = clipped([[nan, 2.0], [3.0]], limit, 0.0)
        assert math.isnan(norm) and all(math.isnan(x) for part in got for x in part)


# ---- what out's rounding does to the gradients -------------------------------------------------------------

def offset_case(dtype, lq, lk, heads, dim):
    """Values and keys far from zero, so that out's rounding is large beside what its gradients are made of: values differ
    by 1 around 64.2, and keys by 1 around 32, which a row's weights do not see.  Queries and out's gradients do not cancel over rows."""
    t = TYPES[dtype]
    q = (0.25 + 0.1 * normal(1, lq, heads, dim)).to(t)
    k, v = (32 + normal(2, lk, 1, dim)).to(t), (64.2 + normal(3, lk, 1, dim)).to(t)
    return q, k, v, (normal(4, 1, heads, dim) + 0.05 * normal(5, lq, heads, dim)).to(t)


def offset_reference(q, k, v, do, scale):
    """dq, dk in 64 bits for one sequence both ways, their tolerances where delta's error has been taken off, and what it would leave
    per unit of it.

    ds~ = (ds - p d) (1 + u), d the error of delta by the rounded out and its rounded weights (2 u of their sizes).  By rows
    sum ds~ is taken off times sum p~ k: what is left of d is multiplied by what p~ and its sum are off by (u and 32-bit errors),
    and roundings act on k's distance from its weighted mean.  By keys d is replaced by the 32-bit errors of the sum that finds it."""
    u, (n, heads, dim), m = UNIT[q.dtype], q.shape, k.shape[0]
    K, V, a = k[:, 0].double(), v[:, 0].double(), abs(scale)
    r = {x: torch.zeros(y.shape, dtype=torch.float64, device=q.device) for x, y in (("dq", q), ("dk", k), ("left_q", q), ("left_k", k))}
    tol = {"dq": r["dq"].clone(), "dk": r["dk"].clone()}
    for h in range(heads):
        Q, G = q[:, h].double(), do[:, h].double()
        s = scale * Q @ K.t()
        off = (dim + 8) * E * a * (Q.abs() @ K.abs().t())
        lse = torch.logsumexp(s, 1, keepdim=True)
        p = torch.exp(s - lse)
        rel = off + 2 * ((p * off).sum(1, keepdim=True) + (m + 8) * E + 4 * E * lse.abs())
        o, osize = p @ V, p @ V.abs()
        d = (2 * u + (p * rel).sum(1, keepdim=True)) * (G.abs() * osize).sum(1, keepdim=True)
        dp, delta = G @ V.t(), (G * o).sum(1, keepdim=True)
        ds = p * (dp - delta)
        big = ds.abs() + p * d
        edp = (dim + 4) * E * (G.abs() @ V.abs().t() + (G.abs() * osize).sum(1, keepdim=True))
        each = big * (u + rel + 4 * E) + p * edp
        sums = d + each.sum(1, keepdim=True) + (m + 8) * E * big.sum(1, keepdim=True)
        mean = p @ K
        for j in range(dim):
            far = (K[:, j][None] - mean[:, j:j + 1]).abs()
            tol["dq"][:, h, j] = a * ((each * far).sum(1) + (sums * p * (u + rel) * K[:, j].abs()[None]).sum(1)
                                      + 2 * (m + 8) * E * ((big + sums * p) * K[:, j].abs()[None]).sum(1))
        r["dq"][:, h] = scale * ds @ K
        r["left_q"][:, h] = scale * mean
        found = (p * edp + big * (rel + 4 * E)).sum(1, keepdim=True) + (m + 8) * E * big.sum(1, keepdim=True) + 4 * E * delta.abs()
        r["dk"][:, 0] += scale * ds.t() @ Q
        r["left_k"][:, 0] += scale * p.t() @ Q
        more = (n * heads + 8) * E
        tol["dk"][:, 0] += a * (ds.abs() * (u + rel + 4 * E + more) + p * (edp + found)).t() @ Q.abs()
        if q.dtype == torch.float16:  # what its powers of two lose of a row's or key's largest one
            tol["dq"][:, h] += 2.0 ** -39 * a * big.amax(1, keepdim=True) * K.abs().sum(0)
            tol["dk"][:, 0] += 2.0 ** -39 * a * big.amax(0)[:, None] * Q.abs().sum(0)
    tol["dq"] += u * r["dq"].abs() + TINY[q.dtype]
    tol["dk"] += u * r["dk"].abs() + TINY[q.dtype]
    return r, tol


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lq,lk", [(64, 64), (20, 1500), (300, 100)])
def test_the_rounding_of_out_is_taken_off_the_gradients(tr, dtype, lq, lk):
    """In one workgroup's pass over the keys, and in parts of them (20 rows of 1500 keys)."""
    print("rounding of out", dtype, lq, lk, flush=True)
    heads, dim, scale = 2, 64, 0.125
    q, k, v, do = offset_case(dtype, lq, lk, heads, dim)
    out, _, dq, dk, _ = attention_both(tr, q, k, v, do, bounds([lq]), bounds([lk]), False, scale)
    want, tol = offset_reference(q, k, v, do, scale)
    within(dq, want["dq"], tol["dq"])
    within(dk, want["dk"], tol["dk"])
    # left in, or taken off twice or the wrong way, it would pass the tolerance somewhere
    exact = torch.stack([torch.softmax(scale * q[:, h].double() @ k[:, 0].double().t(), 1) @ v[:, 0].double() for h in range(heads)], 1)
    delta = (do.double() * (out.double() - exact)).sum(2, keepdim=True)
    assert ((delta * want["left_q"]).abs() > 2 * tol["dq"]).any()
    if dtype == "bf16":
        assert (float(delta.abs().median()) * want["left_k"].abs() > 2 * tol["dk"]).any()


def test_arrays_of_other_kinds_among_gradients_are_refused(tr):
    import numpy as np

    import vector_hip as vh

    g, o = normal(1, 50), normal(2, 50)
    for other in (g.cpu(), g.to("meta"), np.zeros(50, np.float32), [1.0], None):
        for call in (lambda: tr.gradient_norm([g, other]), lambda: tr.clip_gradients([g, other], 1.0), lambda: tr.clip_gradients([g, other], 1.0, out=[o, o]),  # noqa: B023
                     lambda: tr.clip_gradients([g], 1.0, out=[other])):  # noqa: B023
            with pytest.raises(vh.InvalidConfig):
                call()
