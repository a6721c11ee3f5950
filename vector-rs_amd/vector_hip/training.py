"""vector_hip.training -- operators that train the vectors which the engines search.

* ``layer_norm`` / ``layer_norm_backward``       the last layer before an embedding
* ``softmax_xent`` / ``softmax_xent_grad``       cross entropy against every row of a table, and its gradients
* ``orthogonalize``                              Newton-Schulz steps on update matrices

They have no counterpart in the reference.  Arguments are arrays in the memory of one GPU: objects with the
tensor interface ``data_ptr() / dtype / shape / stride() / device / new_empty()`` (torch's, which this module
does not need itself: outputs and working memory come from the arguments' own ``new_empty``).  Element types
are float32, float16 and bfloat16.  The last dimension is contiguous; rows may be any distance apart.

A call enqueues its work on the current stream of its arguments' device and returns without waiting, as
other operations on such arrays do.  Wrong arguments raise ``InvalidConfig``; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import sys
from typing import Optional, Tuple

from . import InvalidConfig, _check, _lib, _sig, _sz

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

_codes = {}   # dtype object -> code
_tensors = {}  # dtype class -> (library, its float32, uint8 and int64)


def _code(dtype) -> int:
    c = _codes.get(dtype)
    if c is None:
        c = _NAMES.get(str(dtype))
        if c is None:
            raise InvalidConfig(f"element type {dtype} is not float32, float16 or bfloat16")
        _codes[dtype] = c
    return c


def _library(a):
    """The library that the caller's arrays come from, with the types that calls make outputs of."""
    kind = type(a.dtype)
    got = _tensors.get(kind)
    if got is None:
        lib = sys.modules[kind.__module__]
        got = _tensors[kind] = (lib, lib.float32, lib.uint8, lib.int64)
    return got


def _on_gpu(name, a):
    if not hasattr(a, "data_ptr") or not hasattr(a, "new_empty"):
        raise InvalidConfig(f"{name} is not a GPU array")
    if a.device.type != "cuda":
        raise InvalidConfig(f"{name} is not in GPU memory")


def _rows2(name, a, like=None) -> int:
    """Checks a matrix of contiguous rows; its distance between rows."""
    _on_gpu(name, a)
    if a.dim() != 2:
        raise InvalidConfig(f"{name} must have two dimensions")
    if like is not None and (a.dtype != like.dtype or a.device != like.device):
        raise InvalidConfig(f"{name} must have the type and the device of the other rows")
    ld, one = a.stride()
    n, d = a.shape
    if one != 1 and d > 1:
        raise InvalidConfig(f"the values of a row of {name} must be contiguous")
    if n <= 1:
        return d
    if ld < d:
        raise InvalidConfig(f"rows of {name} overlap")
    return ld


def _vector(name, a, n, like, dtype=None):
    _on_gpu(name, a)
    if a.dim() != 1 or a.shape[0] != n or (n > 1 and a.stride(0) != 1):
        raise InvalidConfig(f"{name} must hold {n} contiguous values")
    if a.device != like.device:
        raise InvalidConfig(f"{name} is on another device")
    if dtype is not None and a.dtype != dtype:
        raise InvalidConfig(f"{name} must be of {dtype}")


def _ptr(a) -> Optional[int]:
    return None if a is None else a.data_ptr()


def _place(lib, a) -> Tuple[int, int]:
    s = lib.cuda.current_stream(a.device)
    return s.device_index, s.cuda_stream


def _params(x, weight, bias):
    """Checks a layer norm's parameters; the code of their type."""
    code = None
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        _vector(name, p, x.shape[1], x)
        c = _code(p.dtype)
        if code is not None and c != code:
            raise InvalidConfig("weight and bias must have the same type")
        code = c
    return _param_code(code, x)


def _param_code(code, x) -> int:
    if code is None:
        return _code(x.dtype)
    if code not in (F32, _code(x.dtype)):
        raise InvalidConfig("parameters must have the rows' type or float32")
    return code


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """(y, mean, rstd): y = (x - mean) rstd weight + bias over the last dimension of x [rows, dim], with
    rstd = 1 / sqrt(variance + eps).  y has x's type; the statistics are float32."""
    ldx = _rows2("x", x)
    lib, f32, _, _ = _library(x)
    rows, dim = x.shape
    params = _params(x, weight, bias)
    y, mean, rstd = x.new_empty((rows, dim)), x.new_empty((rows,), dtype=f32), x.new_empty((rows,), dtype=f32)
    ordinal, stream = _place(lib, x)
    _check(_lib.vhip_layer_norm(ordinal, _code(x.dtype), params, x.data_ptr(), rows, dim, ldx, _ptr(weight), _ptr(bias),
                                eps, y.data_ptr(), dim, mean.data_ptr(), rstd.data_ptr(), stream))
    return y, mean, rstd


def layer_norm_backward(dy, x, weight, mean, rstd, param_dtype=None):
    """(dx, dweight, dbias) from the gradient of layer_norm's y, its x and weight (or None) and its statistics.
    The parameters' gradients have the weight's type; without a weight `param_dtype` (x's type by default)."""
    ldx, lddy = _rows2("x", x), _rows2("dy", dy, x)
    lib, f32, u8, _ = _library(x)
    rows, dim = x.shape
    if tuple(dy.shape) != (rows, dim):
        raise InvalidConfig("dy must have the shape of x")
    _vector("mean", mean, rows, x, f32)
    _vector("rstd", rstd, rows, x, f32)
    params = _params(x, weight, None)
    ptype = weight.dtype if weight is not None else x.dtype
    if weight is None and param_dtype is not None:
        ptype, params = param_dtype, _param_code(_code(param_dtype), x)
    dx, dweight, dbias = x.new_empty((rows, dim)), x.new_empty((dim,), dtype=ptype), x.new_empty((dim,), dtype=ptype)
    need = _lib.vhip_layer_norm_backward_workspace(rows, dim)
    ws = x.new_empty((need,), dtype=u8)
    ordinal, stream = _place(lib, x)
    _check(_lib.vhip_layer_norm_backward(ordinal, _code(x.dtype), params, dy.data_ptr(), lddy, x.data_ptr(), ldx,
                                         _ptr(weight), mean.data_ptr(), rstd.data_ptr(), rows, dim, dx.data_ptr(), dim,
                                         dweight.data_ptr(), dbias.data_ptr(), ws.data_ptr(), need, stream))
    return dx, dweight, dbias


def _xent_args(h, table, target, bias, row_weight):
    ldh, ldt = _rows2("h", h), _rows2("table", table, h)
    lib, f32, u8, i64 = _library(h)
    rows, dim = h.shape
    if table.shape[1] != dim:
        raise InvalidConfig(f"rows have {dim} elements, the table's have {table.shape[1]}")
    if table.shape[0] == 0:
        raise InvalidConfig("the table is empty")
    _vector("target", target, rows, h, i64)
    if bias is not None:
        _vector("bias", bias, table.shape[0], h, f32)
    if row_weight is not None:
        _vector("row_weight", row_weight, rows, h, f32)
    return ldh, ldt, lib, f32, u8


def softmax_xent(h, table, target, scale: float = 1.0, bias=None):
    """(loss, lse) of the rows of h [rows, dim] against every row of table [n, dim], float32 each:
    z = scale h table^T + bias, lse = log sum exp z, loss = lse - z[target].  target is int64; a negative one
    has loss 0.  bias (float32, constant) may hold -inf, which leaves an entry out."""
    ldh, ldt, lib, f32, u8 = _xent_args(h, table, target, bias, None)
    rows, dim = h.shape
    n, code = table.shape[0], _code(h.dtype)
    loss, lse = h.new_empty((rows,), dtype=f32), h.new_empty((rows,), dtype=f32)
    need = _lib.vhip_softmax_xent_workspace(code, rows, n, dim, 0)
    ws = h.new_empty((need,), dtype=u8)
    ordinal, stream = _place(lib, h)
    _check(_lib.vhip_softmax_xent(ordinal, code, h.data_ptr(), rows, ldh, table.data_ptr(), n, ldt, dim,
                                  target.data_ptr(), _ptr(bias), scale, loss.data_ptr(), lse.data_ptr(), ws.data_ptr(),
                                  need, stream))
    return loss, lse


def softmax_xent_grad(h, table, target, row_weight=None, scale: float = 1.0, bias=None):
    """(loss, lse, dh, dtable): softmax_xent with the gradients of sum(row_weight * loss) for h and the table,
    in their type.  row_weight (float32) is 1 everywhere by default; 1 / (number of targets) gives the mean."""
    ldh, ldt, lib, f32, u8 = _xent_args(h, table, target, bias, row_weight)
    rows, dim = h.shape
    n, code = table.shape[0], _code(h.dtype)
    loss, lse = h.new_empty((rows,), dtype=f32), h.new_empty((rows,), dtype=f32)
    dh, dtable = h.new_empty((rows, dim)), h.new_empty((n, dim))
    need = _lib.vhip_softmax_xent_workspace(code, rows, n, dim, 1)
    ws = h.new_empty((need,), dtype=u8)
    ordinal, stream = _place(lib, h)
    _check(_lib.vhip_softmax_xent_grad(ordinal, code, h.data_ptr(), rows, ldh, table.data_ptr(), n, ldt, dim,
                                       target.data_ptr(), _ptr(bias), _ptr(row_weight), scale, loss.data_ptr(),
                                       lse.data_ptr(), dh.data_ptr(), dim, dtable.data_ptr(), dim, ws.data_ptr(), need,
                                       stream))
    return loss, lse, dh, dtable


def orthogonalize(update, steps: int = 5, coefficients=(3.4445, -4.7750, 2.0315), eps: float = 1e-7):
    """`steps` Newton-Schulz steps on update [rows, cols], or on each matrix of a stack [count, rows, cols]:
    X = M / (|M| + eps); A = X X^T; X <- a X + (b A + c A A) X.  The result has the update's type."""
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
    lib, _, u8, _ = _library(update)
    out = update.new_empty(tuple(update.shape))
    need = _lib.vhip_orthogonalize_workspace(count, rows, cols)
    ws = update.new_empty((need,), dtype=u8)
    ordinal, stream = _place(lib, update)
    _check(_lib.vhip_orthogonalize(ordinal, _code(update.dtype), update.data_ptr(), count, rows, cols, ld,
                                   st[0] if update.dim() == 3 else 0, steps, a, b, c, eps, out.data_ptr(), cols,
                                   rows * cols, ws.data_ptr(), need, stream))
    return out
