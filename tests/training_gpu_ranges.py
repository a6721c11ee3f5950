"""Training operators: values of any size in places that do not count, rows of sizes far apart, limits of sizes
and coefficients, and the kernels that only larger calls reach.  Definitions and tolerances are those of
training_gpu_cases.py; what is new is derived where it stands.

test_training_ranges_gpu.py runs this file in a process of its own, where torch is imported before the library."""
import math

import pytest

torch = pytest.importorskip("torch")

import training_gpu_cases as base  # noqa: E402
from training_gpu_cases import E, TINY, TYPES, UNIT, normal, tr, within, xent_check, xent_inputs, xent_reference  # noqa: E402,F401

pytestmark = pytest.mark.gpu


# ---- what does not count, whatever it holds ---------------------------------------------------------------

def same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(20, 96), (100, 96), (150, 300), (150, 640)])
@pytest.mark.parametrize("value", [1e30, -1e6, 3e4, math.inf, math.nan])
def test_values_of_entries_that_are_left_out(tr, dtype, rows, dim, value):
    """A bias of -inf: the call is what it is with zeros there, to the last bit."""
    h, w, y = xent_inputs(rows, 700, dim, dtype)
    bias = 0.3 * normal(5, 700)
    out = torch.rand(700, device="cuda", generator=base.gen(6)) < 0.2
    out[y] = False
    bias[out] = -math.inf
    w[out] = 0.0
    want = tr.softmax_xent_grad(h, w, y, scale=2.0, bias=bias)
    want_loss = tr.softmax_xent(h, w, y, scale=2.0, bias=bias)
    xent_check(want, h, w, y, 2.0, bias)
    w[out] = value
    same(tr.softmax_xent_grad(h, w, y, scale=2.0, bias=bias), want)
    same(tr.softmax_xent(h, w, y, scale=2.0, bias=bias), want_loss)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(20, 96), (100, 96), (150, 300), (150, 640)])
@pytest.mark.parametrize("value", [1e30, -1e6, 3e4, math.inf, math.nan])
def test_values_of_rows_without_a_target(tr, dtype, rows, dim, value):
    """A negative target: everything but that row's lse is what it is with zeros there, to the last bit, and the
    lse is that of the row's values."""
    h, w, y = xent_inputs(rows, 700, dim, dtype)
    y[2::7] = -1
    rest = y >= 0
    h[~rest] = 0.0
    loss, lse, dh, dw = tr.softmax_xent_grad(h, w, y, scale=2.0)
    xent_check((loss, lse, dh, dw), h, w, y, 2.0)
    h[~rest] = value * (1 + 0.1 * normal(8, int((~rest).sum()), dim)).to(h.dtype)
    loss2, lse2, dh2, dw2 = tr.softmax_xent_grad(h, w, y, scale=2.0)
    same((loss2, lse2[rest], dh2, dw2), (loss, lse[rest], dh, dw))
    if torch.isfinite(h).all() and abs(value) < 1e8:
        hd, wd = h[~rest].double(), w.double()
        z = hd @ wd.t() * 2.0
        want = torch.logsumexp(z, 1)
        # a logit's sum of dim products and its roundings (32-bit values to 2^-22 each), as in xent_check
        zerr = ((dim + 24) * E * 2.0 * (hd.abs() @ wd.abs().t()) + 4 * E * z.abs()).max(1).values
        within(lse2[~rest], want, zerr + 64 * E + 4 * E * want.abs())


# ---- rows of sizes far apart ------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,dim", [(20, 96), (100, 96), (150, 300)])
@pytest.mark.parametrize("power", [-60, 12, 20, 30])
def test_one_row_far_larger_than_the_others(tr, rows, dim, power):
    """In 32 bits each row's loss has the accuracy of its own values."""
    h, w, y = xent_inputs(rows, 700, dim, "f32")
    h[rows // 2] *= 2.0 ** power
    xent_check(tr.softmax_xent_grad(h, w, y, scale=2.0), h, w, y, 2.0)
    xent_check((*tr.softmax_xent(h, w, y, scale=2.0), None, None), h, w, y, 2.0)
    h *= 2.0 ** -100
    xent_check((*tr.softmax_xent(h, w * 2.0 ** 100, y, scale=2.0), None, None), h, w * 2.0 ** 100, y, 2.0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(20, 96), (100, 96), (150, 300), (90, 640)])
def test_row_weights_far_apart(tr, dtype, rows, dim, monkeypatch):
    """Each row's gradient has the accuracy of its own weight: here over 2^26 (2^60 in 32 bits and bfloat16)."""
    h, w, y = xent_inputs(rows, 500, dim, dtype)
    h, w = h / 32, w * 32
    low, high = (-16, 10) if dtype == "f16" else (-40, 20)
    weight = torch.exp2(torch.linspace(low, high, rows, device="cuda"))[torch.randperm(rows, device="cuda", generator=base.gen(3))]
    _, _, rdh, rdw, g, z, hd, wd = xent_reference(h, w, y, 1.0, None, weight)
    t = h.dtype
    # the relative error of p and of 1 - p: that of the logits and the sum; then G's rounding (two planes in 32
    # bits), the sum's chain and the planes of the table.  What G's smallest step leaves out is below
    # 2^-24 / 2^13 of the row's largest value a value of the row, in float16; a plane more in 32 bits.
    per = (dim + 8 if t != torch.float32 else dim + 24) * E
    zerr = (per * (hd.abs() @ wd.abs().t()) + 4 * E * z.abs()).max(1).values
    unit = UNIT[t] if t != torch.float32 else 2.0 ** -22
    rel = 4 * (zerr + 128 * E) + unit + (500 + 32) * E + 2.0 ** -22
    least = 2.0 ** -37 * g.abs().max(1, keepdim=True).values * wd.abs().sum(0) if t != torch.bfloat16 else 0.0
    aw = wd.abs()
    tol = UNIT[t] * rdh.abs() + TINY[t] + rel[:, None] * (g.abs() @ aw) + least + 2.0 ** -38 * aw.max() * g.abs().sum(1, keepdim=True)
    within(tr.softmax_xent_grad(h, w, y, weight)[2], rdh, tol)
    xent_check(tr.softmax_xent_grad(h, w, y, weight), h, w, y, 1.0, None, weight)
    monkeypatch.setenv("VHIP_XENT_PIECE_BYTES", "1")
    within(tr.softmax_xent_grad(h, w, y, weight)[2], rdh, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_row_weights_that_grow_from_piece_to_piece(tr, dtype, monkeypatch):
    """Pieces of 256 rows whose weights differ by 2^12 from one to the next, and a last piece without any."""
    h, w, y = xent_inputs(900, 500, 96, dtype)
    weight = torch.exp2(12.0 * (torch.arange(900, device="cuda") // 256) - 24)
    y[768:] = -1
    monkeypatch.setenv("VHIP_XENT_PIECE_BYTES", "1")
    xent_check(tr.softmax_xent_grad(h, w, y, weight), h, w, y, 1.0, None, weight)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(20, 96), (100, 96), (90, 640)])
def test_rows_of_zeros_and_rows_without_a_loss(tr, dtype, rows, dim):
    """Rows of zeros, beside them rows whose loss is nothing, and rows of both sizes that have no weight."""
    h, w, y = xent_inputs(rows, 500, dim, dtype)
    weight = torch.rand(rows, device="cuda", generator=base.gen(9)) / rows
    h[3::5] = 0.0
    h[4::5] = 30 * w[y[4::5]]
    weight[::9] = 0.0
    xent_check(tr.softmax_xent_grad(h, w, y, weight, scale=2.0), h, w, y, 2.0, None, weight)
    h[:] = 0.0
    xent_check(tr.softmax_xent_grad(h, w, y, weight, scale=2.0), h, w, y, 2.0, None, weight)
    h[:] = 30 * w[y]
    got = tr.softmax_xent_grad(h, w, y, weight, scale=2.0)
    xent_check(got, h, w, y, 2.0, None, weight)
    assert not got[0].any() and not got[2].any() and not got[3].any()


@pytest.mark.parametrize("rows,dim", [(20, 96), (100, 96), (150, 300), (300, 640)])
@pytest.mark.parametrize("power", [12, 20, 30, 60])
@pytest.mark.parametrize("pieces", [False, True])
def test_one_entry_far_larger_than_the_others(tr, rows, dim, power, pieces, monkeypatch):
    """An entry that no row comes near (its logits are below -2^power): everything is as without it."""
    if pieces:
        monkeypatch.setenv("VHIP_XENT_PIECE_BYTES", "1")
    h, w, y = xent_inputs(rows, 700, dim, "f32")
    y = torch.where(y == 5, 6, y)
    h[:, 0], w[5] = 1.0, 0.0
    w[5, 0] = -2.0 ** power
    w[9:300:7] *= 2.0 ** -14
    bias = 0.3 * normal(5, 700)
    keep = torch.arange(700, device="cuda") != 5
    at = y - (y > 5).long()
    loss, lse, dh, dw = tr.softmax_xent_grad(h, w, y, scale=2.0, bias=bias)
    few = w[keep].contiguous()
    off = bias[keep].contiguous()
    _, _, rdh, _, g, *_ = xent_reference(h, few, at, 2.0, off)
    want = tr.softmax_xent_grad(h, few, at, scale=2.0, bias=off)
    xent_check((loss, lse, want[2], dw[keep].contiguous()), h, few, at, 2.0, off)
    assert not dw[5].any()
    xent_check((loss, lse, dh, want[3]), h, few, at, 2.0, off)
    # 32-bit operands' G and sums as in xent_check, for logits below 32, and G's smallest step in every entry
    a = few.double().abs()
    within(dh, rdh, 2.0 ** -16 * (g.abs() @ a) + 2.0 ** -36 * g.abs().max(1, keepdim=True).values * a.sum(0) + 2.0 ** -40)
    xent_check((*tr.softmax_xent(h, w, y, scale=2.0, bias=bias), None, None), h, few, at, 2.0, off)


@pytest.mark.parametrize("rows,dim", [(20, 96), (100, 96), (150, 300), (300, 640)])
@pytest.mark.parametrize("pieces", [False, True])
def test_entries_of_sizes_far_apart(tr, rows, dim, pieces, monkeypatch):
    """Entries from 2^-60 of the largest to the largest, zeros among them."""
    if pieces:
        monkeypatch.setenv("VHIP_XENT_PIECE_BYTES", "1")
    h, w, y = xent_inputs(rows, 700, dim, "f32")
    w *= torch.exp2(-60.0 * torch.rand(700, 1, device="cuda", generator=base.gen(4)) ** 2)
    w[::11] = 0.0
    xent_check(tr.softmax_xent_grad(h, w, y, scale=2.0), h, w, y, 2.0)
    xent_check((*tr.softmax_xent(h, w, y, scale=2.0), None, None), h, w, y, 2.0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(20, 96), (100, 96), (150, 640)])
@pytest.mark.parametrize("value", [math.nan, math.inf, 6e4])
def test_values_of_rows_whose_target_is_left_out(tr, dtype, rows, dim, value):
    """Loss +inf and no part in the gradients, whatever the row holds."""
    h, w, y = xent_inputs(rows, 700, dim, dtype)
    bias = torch.zeros(700, device="cuda")
    y[:] = y % 699
    y[3::9] = 699
    bias[699] = -math.inf
    gone = y == 699
    want = tr.softmax_xent_grad(h, w, y, bias=bias)
    xent_check(want, h, w, y, 1.0, bias)
    assert (want[0][gone] == math.inf).all() and not want[2][gone].any()
    h[gone] = value
    loss, lse, dh, dw = tr.softmax_xent_grad(h, w, y, bias=bias)
    same((loss, lse[~gone], dh, dw), (want[0], want[1][~gone], want[2], want[3]))


# ---- limits ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_rows_than_an_operand_of_a_product_may_have(tr, dtype):
    """Past 2^22 (16 bits: 2^23) rows the products' limit on K and not the size of G makes the pieces."""
    rows, table, dim = (1 << 22) + 1000 if dtype == "f32" else (1 << 23) + 1000, 90, 8
    h, w, y = xent_inputs(rows, table, dim, dtype)
    loss, lse, dh, dw = tr.softmax_xent_grad(h, w, y, scale=2.0)
    for part in (slice(0, 128), slice(rows - 128, rows)):
        xent_check((loss[part], lse[part], None, None), h[part], w, y[part], 2.0)
    step, total, size = 1 << 20, torch.zeros(table, dim, dtype=torch.float64, device="cuda"), 0.0
    for i in range(0, rows, step):
        z = (h[i:i + step].double() @ w.double().t()) * 2
        p = torch.softmax(z, 1)
        p[torch.arange(len(z), device="cuda"), y[i:i + step]] -= 1
        p *= 2
        total += p.t() @ h[i:i + step].double()
        size = size + p.abs().t() @ h[i:i + step].double().abs()
        unit = UNIT[h.dtype]
        a = p.abs() @ w.double().abs()
        within(dh[i:i + step], p @ w.double(), 2 * unit * a + (table + 128) * E * a + 2.0 ** -36)
    # G's rounding is at random: over millions of rows it is far below a unit of the absolute sum, as are
    # 32-bit sums in chains of a million
    within(dw, total, 2 * UNIT[h.dtype] * total.abs() + 2.0 ** -10 * size)


# ---- Newton-Schulz --------------------------------------------------------------------------------------

def ns_steps(m, steps, coefficients, eps=1e-7):
    """The definition in 64 bits, with the largest norms that it passes through."""
    a, b, c = coefficients
    x = m.double()
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(steps):
        p = x @ x.t()
        x = a * x + (b * p + c * p @ p) @ x
    return x.t() if tall else x


@pytest.mark.parametrize("shape", [(1, 1), (1, 40), (40, 90), (200, 90), (900, 1000)])
@pytest.mark.parametrize("coefficients,steps", [
    ((25.0, -0.04, 0.0), 2),      # singular values to 25, and back
    ((2.0, -1.5, 0.5), 5),
    ((1.5, -0.5, 0.0), 8),
    ((300.0, 0.0, 0.0), 1),       # B past 255
    ((300.0, -299.0, 0.0), 1),
    ((3000.0, 0.0, 0.0), 2),
    ((10.0, -200.0, 191.0), 1),   # large terms that cancel at one
    ((0.01, 0.0, 0.0), 1),
    ((-2.0, 1.5, -0.5), 3),
])
def test_orthogonalize_with_other_coefficients(tr, shape, coefficients, steps):
    """Steps that take the singular values far from one on their way."""
    m = normal(sum(shape), *shape)
    got, want = tr.orthogonalize(m, steps=steps, coefficients=coefficients).double(), ns_steps(m, steps, coefficients)
    # a step's error is 2^-20 of the sum of its terms' sizes times X, and what was there grows by its largest slope;
    # both bounded over the interval that the singular values can reach
    a, b, c = (abs(v) for v in coefficients)
    s, err = 1.0, 2.0 ** -20
    for _ in range(steps):
        size = a + b * s * s + c * s ** 4
        err = err * (a + 3 * b * s * s + 5 * c * s ** 4) + 2.0 ** -20 * size * s
        s = max(abs(coefficients[0] * v + coefficients[1] * v ** 3 + coefficients[2] * v ** 5) for v in (s * i / 1000 for i in range(1001)))
    assert torch.isfinite(got).all()
    assert float((got - want).norm()) <= err * math.sqrt(min(shape)) + 2.0 ** -23 * float(want.norm())


def test_orthogonalize_refuses_steps_without_a_bound(tr):
    import vector_hip as vh

    m = normal(1, 20, 30)
    for coefficients, steps in (((25.0, 0.0, 0.0), 100), ((1e20, 0.0, 0.0), 1), ((3.0, 40.0, 0.0), 5)):
        with pytest.raises(vh.InvalidConfig):
            tr.orthogonalize(m, steps=steps, coefficients=coefficients)


@pytest.mark.parametrize("eps", [1e-7, 1e-20, 1e-30, 1e-44])
@pytest.mark.parametrize("shape", [(20, 30), (30, 20), (900, 1000)])
def test_orthogonalize_a_zero_matrix(tr, eps, shape):
    """0 / (0 + eps) is 0 for every eps but 0, in a stack beside another matrix too."""
    z = torch.zeros(2, *shape, device="cuda")
    z[1] = normal(3, *shape)
    got = tr.orthogonalize(z, eps=eps)
    assert not got[0].any() and torch.isfinite(got[1]).all() and got[1].any()


# ---- arguments that torch differentiates --------------------------------------------------------------------

def test_arguments_that_require_a_gradient(tr):
    """Outputs have no graph: the forward calls refuse such arguments where a graph is being recorded."""
    import vector_hip as vh

    x, w = normal(1, 6, 32), normal(2, 32)
    h, table, y = xent_inputs(6, 50, 32, "f32")
    for make in (lambda r: tr.layer_norm(r(x), w, w), lambda r: tr.layer_norm(x, r(w), w), lambda r: tr.layer_norm(x, w, r(w)),
                 lambda r: tr.softmax_xent(r(h), table, y), lambda r: tr.softmax_xent(h, r(table), y),
                 lambda r: tr.softmax_xent(h, table, y, bias=r(normal(4, 50))), lambda r: tr.orthogonalize(r(x))):
        leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
        with pytest.raises(vh.InvalidConfig):
            make(leaf)
        want = make(lambda t: t.clone())
        with torch.no_grad():
            got = make(leaf)
        same([got] if torch.is_tensor(got) else got, [want] if torch.is_tensor(want) else want)
        got = make(lambda t: leaf(t).detach())
        same([got] if torch.is_tensor(got) else got, [want] if torch.is_tensor(want) else want)
    # the gradients' calls give what a backward pass wants of them, parameters or not
    grads = tr.softmax_xent_grad(h.clone().requires_grad_(), torch.nn.Parameter(table.clone()), y)
    same(grads, tr.softmax_xent_grad(h, table, y))
    assert not any(t.requires_grad for t in grads)


# ---- kernels that only larger calls reach --------------------------------------------------------------------

@pytest.mark.parametrize("rows,dim", [(1500, 4096), (1100, 2300), (1100, 8192), (530, 16_384), (1300, 1025), (200, 20_000)])
@pytest.mark.parametrize("dtype,params", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
def test_layer_norm_backward_of_many_long_rows(tr, rows, dim, dtype, params):
    """Rows held by 4 and 16 waves, more of them than workgroups, and rows past that."""
    base.test_layer_norm_backward(tr, rows, dim, 0, dtype, params)


@pytest.mark.parametrize("rows,dim,pad", base.LN_SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_layer_norm_scale(tr, rows, dim, pad, dtype):
    """rstd: 64 additions in a chain put the mean off by 64 e mean|x| and the variance by 64 e of itself."""
    x = (normal(1, rows, dim + pad) * 2 + 0.5).to(TYPES[dtype])[:, :dim]
    _, _, rstd = tr.layer_norm(x)
    _, _, rr, _ = base.ln_reference(x, None, None, 1e-5)
    off = 64 * E * 2 * x.double().abs().mean(1) * rr
    within(rstd, rr, rr * (off + off * off + 40 * E))


@pytest.mark.parametrize("rows,table,dim", [(20, 9000, 330), (33, 8192, 100), (40, 9001, 264), (48, 20_000, 65), (49, 8500, 200), (64, 9000, 331),
                                            (17, 8191, 90), (64, 8191, 90)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_softmax_xent_of_few_rows_over_longer_tables(tr, rows, table, dim, dtype):
    """Turns of 16 and of 32 entries, one to four blocks of rows."""
    h, w, y = xent_inputs(rows, table, dim, dtype)
    bias = 0.3 * normal(5, table)
    out = int(y[0]) - 1
    bias[out] = -math.inf
    y = torch.where(y == out % table, int(y[0]), y)
    xent_check((*tr.softmax_xent(h, w, y, scale=2.0), None, None), h, w, y, 2.0)
    xent_check(tr.softmax_xent_grad(h, w, y, scale=2.0, bias=bias), h, w, y, 2.0, bias)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_softmax_xent_of_more_rows_than_a_join_takes_by_fours(tr, dtype):
    h, w, y = xent_inputs(9001, 300, 40, dtype)
    weight = torch.rand(9001, device="cuda", generator=base.gen(9)) / 9001
    xent_check(tr.softmax_xent_grad(h, w, y, weight, scale=2.0), h, w, y, 2.0, None, weight)


def pairs_model(m, steps, eps=1e-7):
    """The steps with X, A and B rounded to pairs of float16 (22 bits) where they are held so, in 64 bits else:
    how far that alone takes the result from the definition."""
    def pair(x, scale):
        hi = (x * scale).half().double()
        return (hi + (x * scale - hi).half().double()) / scale

    a, b, c = base.NS
    x = m.double()
    x = x / (x.norm() + eps)
    x = x.t() if x.shape[0] > x.shape[1] else x
    x = pair(x, 1024.0)
    for i in range(steps):
        p = pair(x @ x.t(), 256.0)
        q = pair(a * torch.eye(len(p), dtype=p.dtype, device=p.device) + b * p + c * p @ p, 256.0)
        x = q @ x
        x = x if i + 1 == steps else pair(x, 1024.0)
    return x if m.shape[0] <= m.shape[1] else x.t()


@pytest.mark.parametrize("rows,cols", [(64, 64), (100, 300), (300, 100), (129, 257), (400, 390), (900, 700), (1500, 1600), (2304, 2200)])
def test_orthogonalize_is_as_near_as_its_pairs(tr, rows, cols):
    """32 bits, 5 steps: no further from the definition than 20 times what holding pairs costs (products drop the
    low halves' product and add in 32 bits, each of about the size of a pair's rounding, over three products a step)."""
    m = 0.01 * normal(rows + cols, rows, cols)
    want = base.ns_reference(m, 5, 1e-7)
    limit = 20 * float((pairs_model(m, 5) - want).norm()) + 4 * E * float(want.norm())
    assert float((tr.orthogonalize(m).double() - want).norm()) <= limit


# ---- rows far from the origin ----------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [2, 3, 49, 300, 769, 1500, 4097, 9001, 20_001])
@pytest.mark.parametrize("value", [1.9, 7.0, 1000.1, 1e4, -12345.67])
def test_layer_norm_of_constant_rows(tr, dim, value):
    """A mean that is off by d makes every deviation d; their own mean takes it out again, to 66 roundings."""
    x = torch.full((5, dim), value, device="cuda")
    y, mean, rstd = tr.layer_norm(x)
    assert float(y.abs().max()) <= 66 * E * 64 * E * abs(value) * 317
    assert float((mean.double() - x[0, 0].double()).abs().max()) <= 2 * E * abs(value)
    assert float((rstd.double() * 1e-5 ** 0.5 - 1).abs().max()) <= 1e-4


@pytest.mark.parametrize("dim", [49, 300, 1500, 4097, 9001, 20_001])
@pytest.mark.parametrize("offset", [100.0, 1e4, -1e5])
def test_layer_norm_of_rows_with_a_large_mean(tr, dim, offset):
    """Deviations from a mean nearby are exact; what is left of the mean's error is 66 roundings of 64 of it."""
    x = normal(1, 40, dim) + offset
    y, mean, rstd = tr.layer_norm(x)
    ry, rm, rr, _ = base.ln_reference(x, None, None, 1e-5)
    left = (66 * E * 64 * E * abs(offset) + 2 * E) * rr
    within(y, ry, left[:, None] + 70 * E * ry.abs() + 2 * E)
    within(mean, rm, 2 * E * rm.abs())
    within(rstd, rr, 70 * E * rr)


@pytest.mark.parametrize("dim", [5, 300, 1500, 9001, 20_001])
def test_layer_norm_of_rows_that_are_not_finite(tr, dim):
    """NaN and infinity reach y and the scale (and the mean), and no other row."""
    x = normal(2, 5, dim)
    x[1, dim // 2] = math.nan
    x[3, dim - 1] = math.inf
    y, mean, rstd = tr.layer_norm(x)
    assert y[1::2].isnan().all() and rstd[1::2].isnan().all() and not mean[1::2].isfinite().any()
    same(tr.layer_norm(x[::2].contiguous()), (y[::2], mean[::2], rstd[::2]))


# ---- the largest and the narrowest sizes -------------------------------------------------------------------

@pytest.mark.parametrize("rows,table,dim,dtype", [(70, 100, 65_536, "f32"), (70, 100, 65_536, "bf16"), (9, 40, 65_536, "f32"), (3, 40, 65_535, "f16"),
                                                  (65, (1 << 22) - 64, 3, "f32"), (65, (1 << 22) - 64, 8, "f16"), (2, (1 << 22) - 65, 5, "bf16")])
def test_softmax_xent_at_the_limits(tr, rows, table, dim, dtype):
    h, w, y = xent_inputs(rows, table, dim, dtype)
    if dim > 1000:
        h = h / 8  # + 0.1 w of the target is a logit of thousands
    xent_check(tr.softmax_xent_grad(h, w, y), h, w, y, 1.0)
    xent_check((*tr.softmax_xent(h, w, y), None, None), h, w, y, 1.0)


@pytest.mark.parametrize("rows,cols", [(1, 65_536), (65_536, 1), (2, 40_000), (65_535, 3), (65_536, 40)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_orthogonalize_at_the_limits(tr, rows, cols, dtype):
    m = (0.01 * normal(5, rows, cols)).to(TYPES[dtype])
    got, want = tr.orthogonalize(m), base.ns_reference(m, 5, 1e-7)
    assert float((got.double() - want).norm()) <= base.ns_tolerance(want, 5, min(rows, cols), 2 * UNIT[m.dtype])


def test_orthogonalize_many_small_matrices(tr):
    m = normal(6, 65_535, 3, 5)
    got = tr.orthogonalize(m)
    for i in (0, 1, 32_768, 65_534):
        want = base.ns_reference(m[i], 5, 1e-7)
        assert float((got[i].double() - want).norm()) <= base.ns_tolerance(want, 5, 3, 2 * E)


@pytest.mark.parametrize("rows,dim", [(3, (1 << 20) + 1), (1, 5_000_000), (300_000, 3), (1_000_000, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer_norm_at_the_limits(tr, rows, dim, dtype):
    """Chains of a thousandth of a long row, and of a 512th of many rows."""
    x = (normal(1, rows, dim) + 0.25).to(TYPES[dtype])
    w, b = 1 + 0.1 * normal(2, dim), 0.1 * normal(3, dim)
    y, mean, rstd = tr.layer_norm(x, w, b)
    ry, rm, rr, xh = base.ln_reference(x, w, b, 1e-5)
    chain = (64 + dim / 1024) * E
    within(rstd, rr, rr * 2 * chain)
    within(y, ry, UNIT[x.dtype] * ry.abs() + TINY[x.dtype] + 4 * chain * (1 + ry.abs()))
    dy = normal(4, rows, dim).to(x.dtype)
    dx, dw, db = tr.layer_norm_backward(dy, x, w, mean, rstd)
    a = dy.double() * w.double()
    size = a.abs() + a.abs().mean(1, keepdim=True) + xh.abs() * (a * xh).abs().mean(1, keepdim=True)
    want = rr[:, None] * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    within(dx, want, UNIT[x.dtype] * want.abs() + TINY[x.dtype] + 8 * chain * rr[:, None] * (1 + xh.abs()) * size)
    rowchain = (rows / 512 + 160) * E
    within(db, dy.double().sum(0), E * dy.double().sum(0).abs() + rowchain * dy.double().abs().sum(0))
    within(dw, (dy.double() * xh).sum(0), E * (dy.double() * xh).sum(0).abs() + 2 * rowchain * (dy.double().abs() * (0.3 * rr[:, None] + xh.abs())).sum(0))
