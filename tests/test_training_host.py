"""Training operators' argument checks at the C ABI, on the CPU: every refusal comes before a device is used."""
import ctypes

import pytest

BAD = -5  # VHIP_ERR_INVALID_CONFIG
F32, F16, BF16 = 0, 1, 2
P = 4096  # a pointer that no call gets to use


@pytest.fixture(scope="module")
def lib():
    from vector_hip import training  # declares the signatures

    return training._lib


def ln(lib, **k):
    a = dict(ordinal=0, dtype=F32, param=F32, x=P, rows=4, dim=8, ldx=8, w=None, b=None, eps=1e-5, y=P, ldy=8, mean=None,
             rstd=None, stream=None)
    a.update(k)
    return lib.vhip_layer_norm(*a.values())


def ln_back(lib, **k):
    a = dict(ordinal=0, dtype=F32, param=F32, dy=P, lddy=8, x=P, ldx=8, w=None, mean=P, rstd=P, rows=4, dim=8, dx=P, lddx=8,
             dw=P, db=P, ws=P, bytes=1 << 20, stream=None)
    a.update(k)
    return lib.vhip_layer_norm_backward(*a.values())


def grad(lib, **k):
    a = dict(ordinal=0, dtype=F32, h=P, rows=4, ldh=8, table=P, n=9, ldt=8, dim=8, target=P, bias=None, weight=None,
             scale=1.0, loss=P, lse=P, dh=P, lddh=8, dt=P, lddt=8, ws=P, bytes=1 << 30, stream=None)
    a.update(k)
    return lib.vhip_softmax_xent_grad(*a.values())


def xent(lib, **k):
    a = dict(ordinal=0, dtype=F32, h=P, rows=4, ldh=8, table=P, n=9, ldt=8, dim=8, target=P, bias=None, scale=1.0, loss=P,
             lse=P, ws=P, bytes=1 << 30, stream=None)
    a.update(k)
    return lib.vhip_softmax_xent(*a.values())


def ortho(lib, **k):
    a = dict(ordinal=0, dtype=F32, inp=P, count=2, rows=4, cols=8, ldi=8, si=32, steps=5, a=3.0, b=-4.0, c=2.0, eps=1e-7,
             out=P, ldo=8, so=32, ws=P, bytes=1 << 30, stream=None)
    a.update(k)
    return lib.vhip_orthogonalize(*a.values())


@pytest.mark.parametrize("call,wrong", [
    (ln, dict(dtype=3)), (ln, dict(dtype=-1)), (ln, dict(param=BF16)), (ln, dict(dtype=F16, param=BF16)), (ln, dict(x=None)),
    (ln, dict(y=None)), (ln, dict(dim=0)), (ln, dict(dim=1 << 30)), (ln, dict(ldx=7)), (ln, dict(ldy=7)), (ln, dict(eps=-1.0)),
    (ln, dict(eps=float("nan"))),
    (ln_back, dict(mean=None)), (ln_back, dict(rstd=None)), (ln_back, dict(dy=None)), (ln_back, dict(lddx=7)),
    (ln_back, dict(ws=None)), (ln_back, dict(bytes=255)), (ln_back, dict(ws=P + 2)),
    (grad, dict(dtype=9)), (grad, dict(h=None)), (grad, dict(target=None)), (grad, dict(table=None)), (grad, dict(n=0)),
    (grad, dict(n=1 << 22)), (grad, dict(dim=0)), (grad, dict(dim=65537, ldh=65537, ldt=65537, lddh=65537, lddt=65537)),
    (grad, dict(ldh=7)), (grad, dict(ldt=7)), (grad, dict(lddh=7)), (grad, dict(lddt=7)), (grad, dict(dh=None, dt=None)),
    (grad, dict(scale=float("inf"))), (grad, dict(scale=float("nan"))), (grad, dict(bytes=100)), (grad, dict(ws=None)),
    (grad, dict(ws=P + 8)), (xent, dict(bytes=100)), (xent, dict(ws=None)), (xent, dict(rows=1 << 30)),
    (ortho, dict(dtype=5)), (ortho, dict(steps=0)), (ortho, dict(steps=101)), (ortho, dict(a=float("nan"))),
    (ortho, dict(eps=-0.1)), (ortho, dict(inp=None)), (ortho, dict(out=None)), (ortho, dict(ldi=7)), (ortho, dict(ldo=7)),
    (ortho, dict(si=31)), (ortho, dict(so=31)), (ortho, dict(ws=None)), (ortho, dict(bytes=64)), (ortho, dict(rows=65537)),
    (ortho, dict(count=65536)),
])
def test_refused(lib, call, wrong):
    assert call(lib, **wrong) == BAD
    assert lib.vhip_last_error()


def test_workspaces_grow_with_what_they_hold(lib):
    size = lib.vhip_softmax_xent_workspace
    assert size(BF16, 100, 5000, 64, 0) < size(BF16, 100, 5000, 64, 1) < size(F32, 100, 5000, 64, 1)
    # the logits' gradient is bounded: eight times the rows do not take eight times the memory
    assert size(BF16, 1 << 16, 131_072, 128, 1) < 2 * size(BF16, 1 << 13, 131_072, 128, 1)
    assert lib.vhip_layer_norm_backward_workspace(1 << 20, 64) == 2 * 4 * 64 * 512
    assert lib.vhip_orthogonalize_workspace(2, 64, 128) > lib.vhip_orthogonalize_workspace(1, 64, 128)


def test_empty_sizes(lib):
    """Workspaces of nothing, and a call without rows, which gets as far as looking for its GPU."""
    for sizes in ((0, 5, 5), (5, 0, 5), (5, 5, 0), (0, 0, 0)):
        assert lib.vhip_softmax_xent_workspace(BF16, *sizes, 1) > 0
    assert lib.vhip_layer_norm_backward_workspace(0, 8) == 0
    lib.vhip_orthogonalize_workspace(0, 0, 0)
    missing = lib.vhip_device_count() + 100
    assert grad(lib, rows=0, ordinal=missing) not in (0, BAD)
    assert ortho(lib, count=0, ordinal=missing) not in (0, BAD)


def test_arrays_on_the_host_are_refused():
    import numpy as np

    import vector_hip as vh
    from vector_hip import training

    class Host(np.ndarray):
        is_cuda = False

    for x in (np.zeros((4, 8), np.float32), np.zeros((4, 8), np.float32).view(Host), [1.0], None):
        for call in (lambda: training.layer_norm(x), lambda: training.orthogonalize(x), lambda: training.softmax_xent(x, x, x),
                     lambda: training.softmax_xent_grad(x, x, x), lambda: training.layer_norm_backward(x, x, None, x, x)):
            with pytest.raises(vh.InvalidConfig):
                call()


@pytest.mark.parametrize("order,refused", [("torch, vector_hip", False), ("vector_hip, torch", True)])
def test_two_hip_runtimes_are_refused(order, refused):
    """torch brings a HIP runtime of its own: loaded after the library's, it makes a second one."""
    import os
    import subprocess
    import sys

    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vector-rs_amd")
    code = (f"import sys; sys.path.insert(0, {pkg!r})\nimport {order}\nfrom vector_hip import training\n"
            "try:\n    training._one_runtime()\n    print('one')\n"
            "except vector_hip.DriverError as e:\n    print('two', e)\n")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    if "No module named 'torch'" in out.stderr:
        pytest.skip("torch is not installed")
    assert out.returncode == 0, out.stderr
    assert out.stdout.startswith("two" if refused else "one"), out.stdout
