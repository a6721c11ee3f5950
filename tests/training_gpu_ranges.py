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
@pytest.mark.parametrize("rows,dim", [(20, 96), (100, 96), (150, 300)])
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
