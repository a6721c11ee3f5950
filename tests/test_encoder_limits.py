"""Arguments of gradient norms that a call does not use, at the C ABI on the CPU."""
import ctypes

import pytest

P, F32, BF16, BAD = 4096, 0, 2, -5


class Array(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("out", ctypes.c_void_p), ("count", ctypes.c_size_t), ("dtype", ctypes.c_int), ("out_dtype", ctypes.c_int)]


@pytest.fixture(scope="module")
def lib():
    from vector_hip import training  # declares the signatures

    return training._lib


@pytest.mark.parametrize("out,out_dtype", [(P + 1, F32), (2 * P, 77), (2 * P, -1), (P, BF16), (None, 99), (P, F32)])
def test_the_norm_alone_does_not_look_at_outputs(lib, out, out_dtype):
    """All checks are passed: the call gets as far as looking for its GPU.  Clipping refuses the same outputs."""
    table = (Array * 2)(Array(P, out, 10, F32, out_dtype), Array(3 * P, out, 10, F32, out_dtype))
    missing = lib.vhip_device_count() + 100
    args = (ctypes.addressof(table), 2)
    assert lib.vhip_gradient_norm(missing, *args, P, P, 1 << 20, None) not in (0, BAD)
    assert lib.vhip_clip_gradients(missing, *args, 1.0, 0.0, P, P, 1 << 20, None) == BAD
