"""vector_hip.training -- operators that train the vectors which the engines search.

* ``layer_norm`` / ``layer_norm_backward``       the last layer before an embedding
* ``softmax_xent`` / ``softmax_xent_grad``       cross entropy against every row of a table, and its gradients
* ``orthogonalize``                              Newton-Schulz steps on update matrices

They have no counterpart in the reference.  Arguments are arrays in the memory of one GPU: objects with the
tensor interface of torch (``data_ptr()``, ``stride()``, ``new_empty()`` and so on), which this module does not
load itself: outputs and working memory come from the arguments' own ``new_empty``.  Element types
are float32, float16 and bfloat16.  The last dimension is contiguous; rows may be any distance apart.

A call enqueues its work on the current stream of its arguments' device and returns without waiting, as
other operations on such arrays do.  Wrong arguments raise ``InvalidConfig``; there is no CPU fallback.

Outputs belong to no graph of automatic differentiation: gradients come from ``layer_norm_backward`` and
``softmax_xent_grad``, which give them for any arguments and are themselves not differentiated.  The other calls
refuse arguments that require a gradient where torch records a graph; call them under ``torch.no_grad()``, or
with ``detach()``.  Tangents of forward-mode differentiation are not carried on either.

Load torch before ``vector_hip``: torch brings a HIP runtime of its own, which this package's library then
uses as well.  In the other order the process holds two, and a stream of the one means nothing to the other;
calls raise ``DriverError`` then.
"""
from __future__ import annotations

import ctypes
import os
import sys

from . import DriverError, InvalidConfig, _check, _lib, _sig, _sz

__all__ = ["layer_norm", "layer_norm_backward", "softmax_xent", "softmax_xent_grad", "orthogonalize"]

F32, F16, BF16 = 0, 1, 2
_NAMES = {"torch.float32": F32, "torch.float16": F16, "torch.bfloat16": BF16}
_int, _f, _p = ctypes.c_int, ctypes.c_float, ctypes.c_void_p

_sig("vhip_layer_norm", _int, _int, _int, _int, _p, _sz, _sz, _sz, _p, _p, _f, _p, _sz, _p, _p, _p)
_sig("vhip_layer_norm_backward_workspace", _sz, _sz, _sz)
_sig("vhip_layer_norm_backward", _int, _int, _int, _int, _p, _sz, _p, _sz, _p, _p, _p, _sz, _sz, _p, _sz, _p, _p, _p,
     _sz, _p)
_sig("vhip_softmax_xent_workspace", _sz, _int, _sz, _sz, _sz, _int)
_sig("vhip_softmax_xent", _int, _int, _int, _p, _sz, _sz, _p, _sz, _sz, _sz, _p, _p, _f, _p, _p, _p, _sz, _p)
_sig("vhip_softmax_xent_grad", _int, _int, _int, _p, _sz, _sz, _p, _sz, _sz, _sz, _p, _p, _p, _f, _p, _p, _p, _sz, _p,
     _sz, _p, _sz, _p)
_sig("vhip_orthogonalize_workspace", _sz, _sz, _sz, _sz)
_sig("vhip_orthogonalize", _int, _int, _int, _p, _sz, _sz, _sz, _sz, _sz, _int, _f, _f, _f, _f, _p, _sz, _sz, _p, _sz,
     _p)

class _Types(dict):
    """dtype object -> code"""

    def __missing__(self, dtype):
        code = _NAMES.get(str(dtype))
        if code is None:
            raise InvalidConfig(f"element type {dtype} is not float32, float16 or bfloat16")
        self[dtype] = code
        return code


_code = _Types()


def _one_runtime():
    """Raises where more than one HIP runtime is loaded into this process."""
    try:
        with open("/proc/self/maps") as maps:
            loaded = {os.path.realpath(line.split()[-1]) for line in maps if "/libamdhip64.so" in line}
    except OSError:
        return
    if len(loaded) > 1:
        raise DriverError(f"two HIP runtimes are loaded ({', '.join(sorted(loaded))}): load torch before vector_hip")


class _Library:
    """What calls need of the library that the caller's arrays come from: the types that they make outputs
    of, and the current stream of a device (by the quicker of the two ways where it has both)."""

    def __init__(self, lib):
        _one_runtime()
        self.f32, self.u8, self.i64 = lib.float32, lib.uint8, lib.int64
        self.records = getattr(lib, "is_grad_enabled", lambda: False)
        current = lib.cuda.current_stream
        self.stream = getattr(lib._C, "_cuda_getCurrentRawStream", lambda index: current(index).cuda_stream)


class _Libraries(dict):
    """dtype class -> _Library"""

    def __missing__(self, kind):
        got = self[kind] = _Library(sys.modules[kind.__module__])
        return got


_library = _Libraries()


def _on_gpu(name, a):
    if not getattr(a, "is_cuda", False):
        raise InvalidConfig(f"{name} is not an array in GPU memory")


def _no_graph(lib, *arrays):
    """Refuses arrays whose gradient would be lost with the outputs' graph."""
    for a in arrays:
        if getattr(a, "requires_grad", False) and lib.records():
            raise InvalidConfig("an argument requires a gradient, and the outputs would have none: "
                                "call this under torch.no_grad() or with detach()")


def _rows2(name, a, like=None) -> int:
    """Checks a matrix of contiguous rows; its distance between rows."""
    if not getattr(a, "is_cuda", False):
        _on_gpu(name, a)
    st = a.stride()
    if len(st) != 2:
        raise InvalidConfig(f"{name} must have two dimensions")
    if like is not None and (a.dtype != like.dtype or a.get_device() != like.get_device()):
        raise InvalidConfig(f"{name} must have the type and the device of the other rows")
    n, d = a.shape
    if st[1] != 1 and d > 1:
        raise InvalidConfig(f"the values of a row of {name} must be contiguous")
    if n <= 1:
        return d
    if st[0] < d:
        raise InvalidConfig(f"rows of {name} overlap")
    return st[0]


def _vector(name, a, n, device, dtype=None) -> int:
    """Checks n contiguous values; their address."""
    if not getattr(a, "is_cuda", False):
        _on_gpu(name, a)
    if a.shape != (n,) or not a.is_contiguous():
        raise InvalidConfig(f"{name} must hold {n} contiguous values")
    if a.get_device() != device:
        raise InvalidConfig(f"{name} is on another device")
    if dtype is not None and a.dtype != dtype:
        raise InvalidConfig(f"{name} must be of {dtype}")
    return a.data_ptr()


def _param_code(dtype, code) -> int:
    c = _code[dtype]
    if c != F32 and c != code:
        raise InvalidConfig("parameters must have the rows' type or float32")
    return c


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """(y, mean, rstd): y = (x - mean) rstd weight + bias over the last dimension of x [rows, dim], with
    rstd = 1 / sqrt(variance + eps).  y has x's type; the statistics are float32."""
    ldx = _rows2("x", x)
    rows, dim = x.shape
    device, code, lib = x.get_device(), _code[x.dtype], _library[type(x.dtype)]
    params, w, b = code, None, None
    if weight is not None:
        w, params = _vector("weight", weight, dim, device), _param_code(weight.dtype, code)
    if bias is not None:
        b, params = _vector("bias", bias, dim, device), _param_code(bias.dtype, code)
        if weight is not None and bias.dtype != weight.dtype:
            raise InvalidConfig("weight and bias must have the same type")
    _no_graph(lib, x, weight, bias)
    y = x.new_empty((rows, dim))
    mean, rstd = x.new_empty((2, rows), dtype=lib.f32).unbind()
    _check(_lib.vhip_layer_norm(device, code, params, x.data_ptr(), rows, dim, ldx, w, b, eps, y.data_ptr(), dim,
                                mean.data_ptr(), rstd.data_ptr(), lib.stream(device)))
    return y, mean, rstd


def layer_norm_backward(dy, x, weight, mean, rstd, param_dtype=None):
    """(dx, dweight, dbias) from the gradient of layer_norm's y, its x and weight (or None) and its statistics.
    The parameters' gradients have the weight's type; without a weight `param_dtype` (x's type by default)."""
    ldx, lddy = _rows2("x", x), _rows2("dy", dy, x)
    rows, dim = x.shape
    if dy.shape != x.shape:
        raise InvalidConfig("dy must have the shape of x")
    device, code, lib = x.get_device(), _code[x.dtype], _library[type(x.dtype)]
    m, r = _vector("mean", mean, rows, device, lib.f32), _vector("rstd", rstd, rows, device, lib.f32)
    w = None
    if weight is not None:
        w, param_dtype = _vector("weight", weight, dim, device), weight.dtype
    elif param_dtype is None:
        param_dtype = x.dtype
    params = _param_code(param_dtype, code)
    dx = x.new_empty((rows, dim))
    dweight, dbias = x.new_empty((2, dim), dtype=param_dtype).unbind()
    need = _lib.vhip_layer_norm_backward_workspace(rows, dim)
    ws = x.new_empty(need, dtype=lib.u8)
    _check(_lib.vhip_layer_norm_backward(device, code, params, dy.data_ptr(), lddy, x.data_ptr(), ldx, w, m, r, rows, dim,
                                         dx.data_ptr(), dim, dweight.data_ptr(), dbias.data_ptr(), ws.data_ptr(), need,
                                         lib.stream(device)))
    return dx, dweight, dbias


def _xent_args(h, table, target, bias):
    ldh, ldt = _rows2("h", h), _rows2("table", table, h)
    rows, dim = h.shape
    n, d = table.shape
    if d != dim:
        raise InvalidConfig(f"rows have {dim} elements, the table's have {d}")
    if n == 0:
        raise InvalidConfig("the table is empty")
    device, lib = h.get_device(), _library[type(h.dtype)]
    y = _vector("target", target, rows, device, lib.i64)
    b = None if bias is None else _vector("bias", bias, n, device, lib.f32)
    return rows, n, dim, ldh, ldt, device, _code[h.dtype], lib, y, b


def softmax_xent(h, table, target, scale: float = 1.0, bias=None):
    """(loss, lse) of the rows of h [rows, dim] against every row of table [n, dim], float32 each:
    z = scale h table^T + bias, lse = log sum exp z, loss = lse - z[target].  target is int64; a negative one
    has loss 0, one past the table NaN.  bias (float32, constant) may hold -inf, which leaves an entry out; a row
    whose target is left out has loss +inf."""
    rows, n, dim, ldh, ldt, device, code, lib, y, b = _xent_args(h, table, target, bias)
    _no_graph(lib, h, table, bias)
    loss, lse = h.new_empty((2, rows), dtype=lib.f32).unbind()
    need = _lib.vhip_softmax_xent_workspace(code, rows, n, dim, 0)
    ws = h.new_empty(need, dtype=lib.u8)
    _check(_lib.vhip_softmax_xent(device, code, h.data_ptr(), rows, ldh, table.data_ptr(), n, ldt, dim, y, b, scale,
                                  loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), need, lib.stream(device)))
    return loss, lse


def softmax_xent_grad(h, table, target, row_weight=None, scale: float = 1.0, bias=None):
    """(loss, lse, dh, dtable): softmax_xent with the gradients of sum(row_weight * loss) for h and the table,
    in their type.  row_weight (float32) is 1 everywhere by default; 1 / (number of targets) gives the mean.
    Rows with a negative target, and those with loss +inf, have no part in the gradients, whatever they hold; a
    target past the table makes its row's gradient and the table's NaN."""
    rows, n, dim, ldh, ldt, device, code, lib, y, b = _xent_args(h, table, target, bias)
    c = None if row_weight is None else _vector("row_weight", row_weight, rows, device, lib.f32)
    loss, lse = h.new_empty((2, rows), dtype=lib.f32).unbind()
    dh, dtable = h.new_empty((rows, dim)), h.new_empty((n, dim))
    need = _lib.vhip_softmax_xent_workspace(code, rows, n, dim, 1)
    ws = h.new_empty(need, dtype=lib.u8)
    _check(_lib.vhip_softmax_xent_grad(device, code, h.data_ptr(), rows, ldh, table.data_ptr(), n, ldt, dim, y, b, c, scale,
                                       loss.data_ptr(), lse.data_ptr(), dh.data_ptr(), dim, dtable.data_ptr(), dim,
                                       ws.data_ptr(), need, lib.stream(device)))
    return loss, lse, dh, dtable


def orthogonalize(update, steps: int = 5, coefficients=(3.4445, -4.7750, 2.0315), eps: float = 1e-7):
    """`steps` Newton-Schulz steps on update [rows, cols], or on each matrix of a stack [count, rows, cols]:
    X = M / (|M| + eps); A = X X^T; X <- a X + (b A + c A A) X.  The result has the update's type.  Coefficients
    that could take a singular value past 2^30 are refused."""
    _on_gpu("update", update)
    if update.dim() not in (2, 3):
        raise InvalidConfig("update must be a matrix or a stack of matrices")
    count = update.shape[0] if update.dim() == 3 else 1
    rows, cols = update.shape[-2:]
    st = update.stride()
    if st[-1] != 1 and cols > 1:
        raise InvalidConfig("the values of a row of update must be contiguous")
    ld = st[-2] if rows > 1 else cols
    if ld < cols:
        raise InvalidConfig("rows of update overlap")
    a, b, c = coefficients
    device, code, lib = update.get_device(), _code[update.dtype], _library[type(update.dtype)]
    _no_graph(lib, update)
    out = update.new_empty(update.shape)
    need = _lib.vhip_orthogonalize_workspace(count, rows, cols)
    ws = update.new_empty(need, dtype=lib.u8)
    _check(_lib.vhip_orthogonalize(device, code, update.data_ptr(), count, rows, cols, ld,
                                   st[0] if update.dim() == 3 else 0, steps, a, b, c, eps, out.data_ptr(), cols,
                                   rows * cols, ws.data_ptr(), need, lib.stream(device)))
    return out
