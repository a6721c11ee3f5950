"""Training operators (layer_norm.hip, softmax_xent.hip, newton_schulz.hip) against their definitions in 64 bits.

Tolerances are bounds of the arithmetic, made from the case's own values: u is half a unit of the output's
type, e = 2^-24 that of a 32-bit operation; a sum of n terms of absolute sum s is held to n e s with n the
longest chain of additions.

test_training_gpu.py runs this file in a process of its own, where torch is imported before the library: torch
brings a HIP runtime, and the other GPU tests want a process with the library's own."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
NS = (3.4445, -4.7750, 2.0315)


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


# ---- layer norm -------------------------------------------------------------------------------------

def ln_reference(x, w, b, eps):
    x = x.double()
    mean = x.mean(1)
    dev = x - mean[:, None]
    rstd = 1 / torch.sqrt((dev * dev).mean(1) + eps)
    xh = dev * rstd[:, None]
    y = xh if w is None else xh * w.double()
    return (y if b is None else y + b.double()), mean, rstd, xh


def ln_tolerance(x, w, b, y, rstd, eps, unit, tiny):
    """64 additions in a chain at most: the mean is off by 64 e mean|x|, and so is every deviation from it
    (plus the value's own rounding); the variance adds 64 e relative, half of it to the scale."""
    ax = x.double().abs()
    dev = 64 * E * (ax + ax.mean(1, keepdim=True))
    aw = 1.0 if w is None else w.double().abs()
    ab = 0.0 if b is None else b.double().abs()
    rel = 64 * E + (dev.mean(1) * rstd) ** 2 + 2 * dev.mean(1) * rstd  # of the scale, from the deviations
    return unit * y.abs() + tiny + (dev * rstd[:, None]) * aw + rel[:, None] * (y.abs() + ab) + 4 * E * (y.abs() + ab)


LN_SHAPES = [(1, 1, 0), (1, 768, 0), (3, 5, 0), (7, 300, 84), (65, 300, 1), (5, 2048, 0), (3, 4096, 8), (2, 8192, 0),
             (2, 9000, 0), (2, 16384, 0), (2, 20_000, 0), (3, 4097, 0), (2, 8193, 0), (1500, 64, 0), (4200, 96, 0)]


@pytest.mark.parametrize("rows,dim,pad", LN_SHAPES)
@pytest.mark.parametrize("dtype,params", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
def test_layer_norm(tr, rows, dim, pad, dtype, params):
    t, p, eps = TYPES[dtype], TYPES[params], 1e-5
    x = (normal(1, rows, dim + pad) * 2 + 0.5).to(t)[:, :dim]
    w, b = (1 + 0.2 * normal(2, dim)).to(p), (0.3 * normal(3, dim)).to(p)
    y, mean, rstd = tr.layer_norm(x, w, b, eps)
    ry, rm, rr, _ = ln_reference(x, w, b, eps)
    assert y.dtype == t and mean.dtype == rstd.dtype == torch.float32
    within(y, ry, ln_tolerance(x, w, b, ry, rr, eps, UNIT[t], TINY[t]))
    within(mean, rm, 65 * E * x.double().abs().mean(1))


@pytest.mark.parametrize("rows,dim,pad", LN_SHAPES)
@pytest.mark.parametrize("dtype,params", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
def test_layer_norm_backward(tr, rows, dim, pad, dtype, params):
    t, p = TYPES[dtype], TYPES[params]
    x = (normal(1, rows, dim + pad) * 2 + 0.5).to(t)[:, :dim]
    w = (1 + 0.2 * normal(2, dim)).to(p)
    dy = normal(4, rows, dim + pad).to(t)[:, :dim]
    _, mean, rstd, _ = ln_reference(x, w, None, 1e-5)
    mean, rstd = mean.float(), rstd.float()
    dx, dw, db = tr.layer_norm_backward(dy, x, w, mean, rstd)
    assert dx.dtype == t and dw.dtype == db.dtype == p
    m, r, g = mean.double()[:, None], rstd.double()[:, None], dy.double()
    xh = (x.double() - m) * r
    a = g * w.double()
    want = r * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    axh = (x.double().abs() + m.abs()) * r  # what xh is made of
    size = r * (a.abs() + a.abs().mean(1, keepdim=True) + axh * (a.abs() * axh).mean(1, keepdim=True))
    within(dx, want, UNIT[t] * want.abs() + TINY[t] + 80 * E * size)
    # a column's sum: every 512th row in a chain at most, 4 of a workgroup and then 512 / 32 of them
    chain = (rows + 511) // 512 + 140
    within(dw, (g * xh).sum(0), UNIT[p] * (g * xh).sum(0).abs() + TINY[p] + chain * E * (g.abs() * axh).sum(0))
    within(db, g.sum(0), UNIT[p] * g.sum(0).abs() + TINY[p] + chain * E * g.abs().sum(0))


def test_layer_norm_gradient_against_differences(tr):
    """A step along a direction changes sum(dy y) by what the gradients say, in 64 bits."""
    rows, dim, eps, h = 9, 50, 1e-3, 1e-4
    x, w, b, dy = normal(1, rows, dim), 1 + 0.2 * normal(2, dim), 0.1 * normal(3, dim), normal(4, rows, dim)
    _, mean, rstd = tr.layer_norm(x, w, b, eps)
    dx, dw, db = tr.layer_norm_backward(dy, x, w, mean, rstd)
    ux, uw, ub = normal(5, rows, dim).double(), normal(6, dim).double(), normal(7, dim).double()
    f = lambda s: (ln_reference(x.double() + s * ux, w.double() + s * uw, b.double() + s * ub, eps)[0] * dy.double()).sum()  # noqa: E731
    slope = (f(h) - f(-h)) / (2 * h)
    said = (dx.double() * ux).sum() + (dw.double() * uw).sum() + (db.double() * ub).sum()
    # 32-bit gradients of 9 x 50 values of order one, and the difference's own h^2
    assert abs(float(slope - said)) <= 1e-4 * math.sqrt(rows * dim)


def test_layer_norm_edges(tr):
    """Constant rows have no variance; a row with NaN or infinity is alone with it; rows far from the origin;
    no weight, no bias, no rows."""
    x = normal(1, 6, 300)
    x[1] = 7.0
    x[2, 5] = math.nan
    x[3, 6] = math.inf
    x[4] += 4096.0
    y, mean, rstd = tr.layer_norm(x)
    assert torch.equal(y[1], torch.zeros_like(y[1])) and abs(float(rstd[1]) - 1e-5 ** -0.5) < 1e-3
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    keep = [0, 1, 4, 5]
    ry, _, rr, _ = ln_reference(x[keep], None, None, 1e-5)
    within(y[keep], ry, ln_tolerance(x[keep], None, None, ry, rr, 1e-5, E, TINY[torch.float32]))
    y, mean, rstd = tr.layer_norm(x[:0])
    assert y.shape == (0, 300) and mean.shape == (0,)
    dx, dw, db = tr.layer_norm_backward(x[:0], x[:0], None, mean, rstd)
    assert dx.shape == (0, 300) and not dw.any() and not db.any()


def test_layer_norm_is_repeatable(tr):
    x, dy = normal(1, 5000, 300), normal(2, 5000, 300)
    _, mean, rstd = tr.layer_norm(x)
    first = tr.layer_norm_backward(dy, x, None, mean, rstd)
    for _ in range(3):
        for a, b in zip(first, tr.layer_norm_backward(dy, x, None, mean, rstd)):
            assert torch.equal(a, b)


# ---- softmax cross entropy -----------------------------------------------------------------------------

def xent_reference(h, w, target, scale, bias=None, weight=None):
    """Loss, lse and gradients in 64 bits, with what does not count left out by hand."""
    rows = h.shape[0]
    out = None if bias is None else bias == -math.inf
    wd = w.double()
    if out is not None:
        wd = wd.masked_fill(out[:, None], 0.0)
    hd = h.double().masked_fill((target < 0)[:, None], 0.0)
    z = hd @ wd.t() * scale
    if bias is not None:
        z = z + bias.double()
    lse = torch.logsumexp(z, 1)
    real = (h.double() @ wd.t() * scale) + (0 if bias is None else bias.double())
    loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
    g = torch.zeros_like(z)
    for t in range(rows):
        y = int(target[t])
        if y < 0:
            continue
        if lse[t] == -math.inf or z[t, y] == -math.inf:
            loss[t] = math.inf
            continue
        # by the other entries, so that 64 bits hold a loss and a 1 - p far below 2^-53
        others = torch.exp(z[t] - z[t, y])
        others[y] = 0.0
        loss[t] = torch.log1p(others.sum())
        if not torch.isfinite(loss[t]):
            loss[t] = lse[t] - z[t, y]
        c = scale * (1.0 if weight is None else float(weight[t]))
        g[t] = c * torch.exp(z[t] - lse[t])
        g[t, y] = 0.0
        g[t, y] = -g[t].sum()
    return loss, torch.logsumexp(real, 1), g @ wd, g.t() @ hd, g, z, hd, wd


def xent_check(got, h, w, target, scale, bias=None, weight=None):
    loss, lse, dh, dw = got
    t = h.dtype
    rl, rs, rdh, rdw, g, z, hd, wd = xent_reference(h, w, target, scale, bias, weight)
    dim = h.shape[1]
    # a logit: dim products of 16-bit values are exact, their 32-bit sum is off by dim e of the absolute sum;
    # 32-bit values are held to 2^-22 each; scale, bias and the difference from the largest add 4 roundings
    per = (dim + 8 if t != torch.float32 else dim + 24) * E
    zabs = (hd.abs() @ wd.abs().t()) * abs(scale)
    zerr = (per * zabs + 4 * E * torch.where(torch.isfinite(z), z.abs(), 0.0)).max(1).values
    live = torch.isfinite(rl)
    # exp by its power of two (24 e relative at arguments up to 16 and less beyond what counts), the sum's chain
    serr = zerr + 64 * E
    within(lse, rs, torch.where(torch.isfinite(rs), serr + 4 * E * rs.abs(), 0.0))
    within(loss, rl, torch.where(live, 2 * serr + 4 * E * torch.where(live, rl.abs(), 0.0), 0.0))
    if dh is None:
        return
    # G: p's relative error is that of its logit and of lse, then the rounding to the operands' type (two
    # planes of float16 for 32 bits); a float16 plane's smallest step is 2^-24 of 2^14 times the largest weight
    c = g.abs() + 0.0
    unit = UNIT[t] if t != torch.float32 else 2.0 ** -22
    top = (torch.ones_like(rl) if weight is None else weight.double().abs()).max() * abs(scale)
    floor = 2.0 ** -36 * top if t != torch.bfloat16 else 0.0
    p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
    cw = (torch.ones_like(rl) if weight is None else weight.double().abs()) * abs(scale)
    counts = live & (target >= 0)
    perr = torch.where(counts[:, None], cw[:, None] * torch.nan_to_num(p) * 2 * (serr + 64 * E)[:, None], 0.0)
    gerr = perr + unit * c + torch.where(counts[:, None], floor, torch.zeros_like(c))
    acc = lambda n: (n + 32) * E  # noqa: E731
    n, m = w.shape[0], h.shape[0]
    aw, ah = wd.abs(), hd.abs()
    slack = 2.0 ** -22 if t == torch.float32 else 0.0  # the planes of the other operand
    within(dh, rdh, UNIT[t] * rdh.abs() + TINY[t] + gerr @ aw + (acc(n) + slack) * (c @ aw) + 2.0 ** -38 * aw.max() * c.sum(1, keepdim=True))
    within(dw, rdw, UNIT[t] * rdw.abs() + TINY[t] + gerr.t() @ ah + (acc(m) + slack) * (c.t() @ ah) + 2.0 ** -38 * ah.max() * c.sum(0)[:, None])


def xent_inputs(rows, table, dim, dtype, seed=0):
    h = normal(seed + 1, rows, dim) / math.sqrt(dim)
    w = normal(seed + 2, table, dim)
    y = torch.randint(0, table, (rows,), device="cuda", generator=gen(seed + 3))
    return (h + 0.1 * w[y]).to(TYPES[dtype]), w.to(TYPES[dtype]), y


XENT_SHAPES = [(1, 1, 1), (1, 5, 3), (2, 1000, 64), (3, 64, 64), (17, 1000, 100), (33, 4099, 256), (129, 300, 65), (256, 257, 128),
               (300, 2049, 320), (130, 70, 768), (700, 1300, 40), (20, 3000, 300), (64, 500, 130), (65, 500, 130),
               (32, 40_000, 24), (50, 129, 1030), (70, 70_000, 520), (260, 515, 390)]


@pytest.mark.parametrize("rows,table,dim", XENT_SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_softmax_xent(tr, rows, table, dim, dtype):
    h, w, y = xent_inputs(rows, table, dim, dtype)
    xent_check((*tr.softmax_xent(h, w, y, scale=2.0), None, None), h, w, y, 2.0)
    weight = torch.rand(rows, device="cuda", generator=gen(9)) / rows
    xent_check(tr.softmax_xent_grad(h, w, y, weight, scale=2.0), h, w, y, 2.0, None, weight)


@pytest.mark.parametrize("rows,table,dim", [(5, 90, 64), (40, 1000, 100), (300, 700, 128), (90, 300, 520)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_softmax_xent_left_out(tr, rows, table, dim, dtype):
    """Entries with a bias of -inf, rows with a negative target and NaN in both places; targets that are left
    out; the lowest finite value as a mask."""
    h, w, y = xent_inputs(rows, table, dim, dtype)
    bias = 0.3 * normal(5, table)
    out = torch.rand(table, device="cuda", generator=gen(6)) < 0.3
    out[y[0]] = False
    out[y[1]] = True
    bias[out] = -math.inf
    bias[int((~out).nonzero()[-1])] = torch.finfo(torch.float32).min
    w[out] = math.nan
    y[2::7] = -100
    h[2::7] = math.nan
    loss, lse, dh, dw = tr.softmax_xent_grad(h, w, y, None, scale=1.5, bias=bias)
    assert loss[1] == math.inf and not dh[1].any() and not dw[out].any()
    assert not loss[2::7].any() and not dh[2::7].any() and torch.isnan(lse[2::7]).all()
    xent_check((loss, lse, dh, dw), h, w, y, 1.5, bias)
    only = tr.softmax_xent(h, w, y, scale=1.5, bias=bias)
    assert torch.equal(only[0], loss) and torch.equal(only[1].isnan(), lse.isnan())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim", [(4, 64), (100, 64), (100, 512)])
def test_softmax_xent_nothing_left(tr, dtype, rows, dim):
    h, w, y = xent_inputs(rows, 130, dim, dtype)
    bias = torch.full((130,), -math.inf, device="cuda")
    loss, lse, dh, dw = tr.softmax_xent_grad(h, w, y, bias=bias)
    assert (loss == math.inf).all() and (lse == -math.inf).all() and not dh.any() and not dw.any()
    y[:] = -1
    loss, _, dh, dw = tr.softmax_xent_grad(h, w, y)
    assert not loss.any() and not dh.any() and not dw.any()
    loss, lse, dh, dw = tr.softmax_xent_grad(h[:0], w, y[:0])
    assert loss.shape == (0,) and dh.shape == (0, dim) and not dw.any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(5, 64), (100, 64), (100, 512)])
def test_softmax_xent_target_past_the_table(tr, dtype, rows, dim):
    h, w, y = xent_inputs(rows, 130, dim, dtype)
    y[3] = 130
    loss, lse, dh, _ = tr.softmax_xent_grad(h, w, y)
    assert torch.isnan(loss[3]) and torch.isnan(dh[3]).all() and torch.isfinite(lse).all()
    rest = [t for t in range(rows) if t != 3]
    assert torch.isfinite(loss[rest]).all() and torch.isfinite(dh[rest]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1e-25, 1e-6, 1.0, 1e6])
@pytest.mark.parametrize("rows,dim", [(20, 64), (70, 64), (70, 512)])
def test_softmax_xent_weights_of_any_size(tr, dtype, size, rows, dim):
    """Row weights far from one, among them a zero and signs, do not cost the gradients their bits."""
    h, w, y = xent_inputs(rows, 500, dim, dtype)
    weight = size * normal(8, rows)
    weight[3] = 0.0
    _, _, dh, dw = tr.softmax_xent_grad(h, w, y, weight)
    rl, _, rdh, rdw, *_ = xent_reference(h, w, y, 1.0, None, weight)
    small = TINY[TYPES[dtype]]
    for got, want in ((dh, rdh), (dw, rdw)):
        over = want.abs().max() > torch.finfo(TYPES[dtype]).max
        if over or want.abs().max() < 1e4 * small:
            continue  # the result itself is outside the type
        norm = float((got.double() - want).norm() / want.norm())
        assert norm <= 4 * max(UNIT[TYPES[dtype]], 2.0 ** -17)
    assert not dh[3].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [9, 150])
def test_softmax_xent_strides_and_values_far_apart(tr, dtype, rows):
    """Columns of wider buffers, at odd offsets; a table whose rows differ by 2^20 in size."""
    big_h, big_w, y = xent_inputs(rows, 600, 131, dtype)
    h, w = big_h[:, 3:131], big_w[:, 2:130]
    assert h.shape[1] == w.shape[1] == 128
    xent_check(tr.softmax_xent_grad(h, w, y, scale=0.5), h, w, y, 0.5)
    w = w.contiguous()
    w[::3] *= 2.0 ** -20
    xent_check(tr.softmax_xent_grad(h, w, y, scale=0.5), h, w, y, 0.5)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [100, 520])
def test_softmax_xent_in_pieces(tr, dtype, dim, monkeypatch):
    """Rows taken 256 at a time give what one piece gives: the same loss, gradients within their rounding."""
    h, w, y = xent_inputs(700, 900, dim, dtype)
    weight = normal(4, 700)
    whole = tr.softmax_xent_grad(h, w, y, weight)
    monkeypatch.setenv("VHIP_XENT_PIECE_BYTES", "1")
    parts = tr.softmax_xent_grad(h, w, y, weight)
    xent_check(parts, h, w, y, 1.0, None, weight)
    within(parts[0], whole[0].double(), 2 * E * 128 * (1 + whole[0].double().abs()))
    xent_check((*tr.softmax_xent(h, w, y), None, None), h, w, y, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,table,dim", [(200, 70_001, 300), (150, 70_000, 137), (300, 45_000, 550), (300, 50_000, 384)])
def test_softmax_xent_gradients_of_narrow_tables(tr, dtype, rows, table, dim, monkeypatch):
    """Columns that fill tiles of 192 better than of 256, in one piece and in pieces of 256 rows."""
    h, w, y = xent_inputs(rows, table, dim, dtype)
    xent_check(tr.softmax_xent_grad(h, w, y), h, w, y, 1.0)
    monkeypatch.setenv("VHIP_XENT_PIECE_BYTES", "1")
    xent_check(tr.softmax_xent_grad(h, w, y), h, w, y, 1.0)


def test_softmax_xent_values_that_differ_in_size_by_entry(tr):
    """Logits of a row spread over hundreds: probabilities down to the smallest that 32 bits hold."""
    h, w, y = xent_inputs(100, 700, 512, "bf16")
    w[::5] *= 40.0
    w[3::64] *= 0.01
    xent_check(tr.softmax_xent_grad(h, w, y, scale=3.0), h, w, y, 3.0)
    xent_check(tr.softmax_xent_grad(h, w, y, scale=-3.0), h, w, y, -3.0)
    xent_check(tr.softmax_xent_grad(h, w, y, scale=0.0), h, w, y, 0.0)


def test_softmax_xent_gradient_against_differences(tr):
    rows, table, dim, s = 20, 150, 30, 1e-4
    h, w, y = xent_inputs(rows, table, dim, "f32")
    weight, bias = normal(5, rows), 0.2 * normal(6, table)
    _, _, dh, dw = tr.softmax_xent_grad(h, w, y, weight, scale=1.3, bias=bias)
    uh, uw = normal(7, rows, dim).double(), normal(8, table, dim).double()
    f = lambda e: (xent_reference(h.double() + e * uh, w.double() + e * uw, y, 1.3, bias)[0] * weight.double()).sum()  # noqa: E731
    slope = (f(s) - f(-s)) / (2 * s)
    said = (dh.double() * uh).sum() + (dw.double() * uw).sum()
    assert abs(float(slope - said)) <= 1e-3 * math.sqrt(rows * dim)


def test_softmax_xent_is_repeatable(tr):
    h, w, y = xent_inputs(300, 5000, 64, "bf16")
    first = tr.softmax_xent_grad(h, w, y)
    for _ in range(3):
        for a, b in zip(first, tr.softmax_xent_grad(h, w, y)):
            assert torch.equal(a, b)


# ---- Newton-Schulz -------------------------------------------------------------------------------------

def ns_reference(m, steps, eps):
    x = m.double()
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(steps):
        p = x @ x.t()
        x = NS[0] * x + (NS[1] * p + NS[2] * p @ p) @ x
    return x.t() if tall else x


def ns_tolerance(want, steps, small, unit):
    """Frobenius norm.  A step rounds its planes and sums to 8 x 2^-22 of X's norm at most, and what it rounds
    grows by 3.9 a later step at most (the largest slope of the step's polynomial up to 1.2); X's norm starts
    at 1 and grows by the coefficient a until every singular value is about one."""
    grown = sum(3.9 ** (steps - 1 - k) * min(3.4445 ** (k + 1), 1.2 * math.sqrt(small)) for k in range(steps))
    return 8 * 2.0 ** -22 * (grown + 3.9 ** steps) + unit * float(want.norm())


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 9), (5, 3), (3, 5), (64, 64), (100, 300), (300, 100), (129, 257), (400, 390), (800, 820), (900, 700)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("steps", [1, 5])
def test_orthogonalize(tr, rows, cols, dtype, steps):
    m = (0.01 * normal(rows + cols, rows, cols)).to(TYPES[dtype])
    got = tr.orthogonalize(m, steps=steps)
    assert got.dtype == m.dtype and got.shape == m.shape
    want = ns_reference(m, steps, 1e-7)
    assert float((got.double() - want).norm()) <= ns_tolerance(want, steps, min(rows, cols), 2 * UNIT[m.dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_orthogonalize_a_stack(tr, dtype):
    """Matrices of a stack, also one with rows and matrices spaced apart, are each what they are alone."""
    big = normal(3, 4, 150, 333).to(TYPES[dtype])
    stack = big[1:, :130, :300]
    got = tr.orthogonalize(stack)
    for i in range(3):
        assert torch.equal(got[i], tr.orthogonalize(stack[i].contiguous()))


@pytest.mark.parametrize("count,rows,cols", [(60, 130, 300), (60, 300, 130), (12, 400, 390), (1, 1500, 1600), (1, 1700, 1410), (1, 900, 2500), (1, 2304, 2200)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("steps", [1, 2, 5])
def test_orthogonalize_many_tiles(tr, count, rows, cols, dtype, steps):
    """Stacks and matrices that take the tiled products."""
    m = (0.01 * normal(rows + cols, count, rows, cols)).to(TYPES[dtype])
    got = tr.orthogonalize(m, steps=steps)
    for i in (0, count - 1):
        want = ns_reference(m[i], steps, 1e-7)
        assert float((got[i].double() - want).norm()) <= ns_tolerance(want, steps, min(rows, cols), 2 * UNIT[m.dtype])


def test_orthogonalize_against_a_large_eps(tr):
    """eps takes part in the scale: a matrix of a thousandth of eps is hardly moved towards one."""
    m = normal(8, 30, 50)
    eps = 1000 * float(m.norm())
    got, want = tr.orthogonalize(m, eps=eps), ns_reference(m, 5, eps)
    assert float((got.double() - want).norm()) <= ns_tolerance(want, 5, 30, 2 * E)


def test_orthogonalize_brings_singular_values_to_one(tr):
    s = torch.linalg.svdvals(tr.orthogonalize(normal(2, 96, 300)).double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1.0, 1e15, 1e25])
def test_orthogonalize_values_of_any_size(tr, size):
    """Squares that 32 bits could not hold; eps is left out, and a zero matrix stays zero."""
    m = size * normal(5, 40, 70)
    got = tr.orthogonalize(m, eps=0.0)
    want = ns_reference(m, 5, 0.0)
    assert float((got.double() - want).norm()) <= ns_tolerance(want, 5, 40, 2 * E)


def test_orthogonalize_edges(tr):
    assert not tr.orthogonalize(torch.zeros(20, 30, device="cuda")).any()
    m = normal(1, 20, 30)
    m[3, 4] = math.nan
    two = torch.stack([m, normal(2, 20, 30)])
    got = tr.orthogonalize(two)
    assert torch.isnan(got[0]).all() and torch.equal(got[1], tr.orthogonalize(two[1]))
    assert tr.orthogonalize(m[:0]).shape == (0, 30) and tr.orthogonalize(two[:0]).shape == (0, 20, 30)


# ---- buffers past 2^32 bytes ---------------------------------------------------------------------------

def test_rows_far_apart(tr):
    """Rows whose last lies more than 2^32 bytes, and 2^31 elements, behind the first."""
    rows, dim, ld = 3000, 64, 1_000_000
    wide = torch.empty(rows, ld, device="cuda", dtype=torch.bfloat16)
    x = wide[:, 8:8 + dim]
    x.copy_(normal(1, rows, dim))
    near = x.contiguous()
    y, mean, rstd = tr.layer_norm(x)
    for a, b in zip((y, mean, rstd), tr.layer_norm(near)):
        assert torch.equal(a, b)
    for a, b in zip(tr.layer_norm_backward(x, x, None, mean, rstd), tr.layer_norm_backward(near, near, None, mean, rstd)):
        assert torch.equal(a, b)
    t = torch.randint(0, rows, (rows,), device="cuda", generator=gen(2))
    for n in (20, 300):
        for a, b in zip(tr.softmax_xent_grad(x[:n], x, t[:n]), tr.softmax_xent_grad(near[:n], near, t[:n])):
            assert torch.equal(a, b)
    assert torch.equal(tr.orthogonalize(x), tr.orthogonalize(near))
    del wide, x


def test_a_gradient_of_many_logits(tr):
    """4.6e9 logits, in pieces of rows: losses by their definition, and a row's gradient as in a small call."""
    rows, table, dim = 2300, 2_000_000, 16
    h, w, y = xent_inputs(rows, table, dim, "bf16")
    weight = torch.ones(rows, device="cuda")
    loss, lse, dh, dw = tr.softmax_xent_grad(h, w, y, weight)
    for at in (0, 1024, rows - 128):
        part = slice(at, at + 128)
        l2, e2, d2, _ = tr.softmax_xent_grad(h[part], w, y[part], weight[part])
        xent_check((loss[part], lse[part], None, None), h[part], w, y[part], 1.0)
        xent_check((l2, e2, None, None), h[part], w, y[part], 1.0)
        within(dh[part], d2.double(), 4 * UNIT[torch.bfloat16] * d2.double().abs() + 1e-4 * d2.double().abs().max())
    # every row's probabilities sum to one: the table's gradient adds up to (what the rows lose) = 0 over entries
    total = dw.double().sum(0)
    assert float(total.abs().max()) <= 2 ** -8 * float(dw.double().abs().sum(0).max())


# ---- streams, graphs, refusals -----------------------------------------------------------------------

def every_call(tr):
    x, dy = normal(1, 200, 300).bfloat16(), normal(2, 200, 300).bfloat16()
    w = normal(3, 300).bfloat16()
    h, table, y = xent_inputs(200, 999, 300, "bf16")
    m = normal(4, 100, 300)

    def run():
        yy, mean, rstd = tr.layer_norm(x, w, w)
        return [yy, mean, rstd, *tr.layer_norm_backward(dy, x, w, mean, rstd), *tr.softmax_xent(h, table, y),
                *tr.softmax_xent_grad(h, table, y), tr.orthogonalize(m)]

    return run


def test_calls_on_another_stream(tr):
    run = every_call(tr)
    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_calls_in_a_graph(tr):
    """Captured once and replayed, with eager work between the replays."""
    run = every_call(tr)
    want = run()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(4):
        for t in got:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        run()
        torch.cuda.synchronize()


def test_refusals(tr):
    import vector_hip as vh

    x, w = normal(1, 4, 30), normal(2, 30)
    h, table, y = xent_inputs(4, 50, 30, "f32")
    bad = [
        lambda: tr.layer_norm(x.cpu()), lambda: tr.layer_norm(x.double()), lambda: tr.layer_norm(x[0]),
        lambda: tr.layer_norm(x.t()), lambda: tr.layer_norm(x, w[:-1]), lambda: tr.layer_norm(x, w.half()),
        lambda: tr.layer_norm(x.half(), w.half(), w), lambda: tr.layer_norm(x, w, eps=-1.0),
        lambda: tr.layer_norm(x, w, eps=math.nan), lambda: tr.layer_norm(x[:, :0]),
        lambda: tr.layer_norm(x[:1].expand(4, 30)), lambda: tr.layer_norm([1.0]),
        lambda: tr.layer_norm_backward(x[:3], x, None, x[:, 0].contiguous(), x[:, 0].contiguous()),
        lambda: tr.layer_norm_backward(x, x, None, x[:, 0], x[:, 0].contiguous()),
        lambda: tr.layer_norm_backward(x, x, None, x[0], x[0]),
        lambda: tr.softmax_xent(h, table[:, :29], y), lambda: tr.softmax_xent(h, table.half(), y),
        lambda: tr.softmax_xent(h, table, y.int()), lambda: tr.softmax_xent(h, table, y[:3]),
        lambda: tr.softmax_xent(h, table[:0], y), lambda: tr.softmax_xent(h, table, y, bias=w),
        lambda: tr.softmax_xent(h, table, y, scale=math.inf), lambda: tr.softmax_xent_grad(h, table, y, w),
        lambda: tr.softmax_xent(h[:, :0], table[:, :0], y),
        lambda: tr.orthogonalize(w), lambda: tr.orthogonalize(x.t()), lambda: tr.orthogonalize(x, steps=0),
        lambda: tr.orthogonalize(x, coefficients=(1.0, math.nan, 0.0)), lambda: tr.orthogonalize(x, eps=-1.0),
        lambda: tr.orthogonalize(x.expand(3, 4, 30)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(vh.InvalidConfig):
            f()
            pytest.fail(f"call {i} was not refused")
