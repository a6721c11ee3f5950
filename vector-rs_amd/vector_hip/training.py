"""vector_hip.training -- operators that train the vectors which the engines search.

* ``layer_norm`` / ``layer_norm_backward``       the last layer before an embedding
* ``softmax_xent`` / ``softmax_xent_grad``       cross entropy against every row of a table, and its gradients
* ``orthogonalize``                              Newton-Schulz steps on update matrices
* ``attention`` / ``attention_backward``         softmax attention over packed sequences with grouped heads
* ``qk_norm_rotary`` / ``..._backward``          norms of queries and keys for each head, turned by position
* ``gradient_norm`` / ``clip_gradients``         the norm of many arrays together, and clipping to a largest one

They have no counterpart in the reference.  Arguments are arrays in the memory of one GPU: objects with the
tensor interface of torch (``data_ptr()``, ``stride()``, ``new_empty()`` and so on), which this module does not
load itself: outputs and working memory come from the arguments' own ``new_empty``.  Element types
are float32, float16 and bfloat16.  The last dimension is contiguous; rows may be any distance apart.

A call enqueues its work on the current stream of its arguments' device and returns without waiting, as
other operations on such arrays do.  Wrong arguments raise ``InvalidConfig``; there is no CPU fallback.

Outputs belong to no graph of automatic differentiation: gradients come from ``softmax_xent_grad`` and the calls
named ``..._backward``, which give them for any arguments and are themselves not differentiated.  The other calls
refuse arguments (``out`` among them) that require a gradient where torch records a graph; call them under ``torch.no_grad()``, or
with ``detach()``.  Tangents of forward-mode differentiation are not carried on either.

Load torch before ``vector_hip``: torch brings a HIP runtime of its own, which this package's library then
uses as well.  In the other order the process holds two, and a stream of the one means nothing to the other;
calls raise ``DriverError`` then.
"""
from __future__ import annotations

import ctypes
import os
import sys
from array import array

from . import DriverError, InvalidConfig, _check, _lib, _sig, _sz

__all__ = ["layer_norm", "layer_norm_backward", "softmax_xent", "softmax_xent_grad", "orthogonalize", "attention",
           "attention_backward", "qk_norm_rotary", "qk_norm_rotary_backward", "gradient_norm", "clip_gradients"]

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


class _Heads(ctypes.Structure):
    _fields_ = [("data", _p), ("token", _sz), ("head", _sz)]


_h = ctypes.POINTER(_Heads)
_shape = [_sz] * 6  # tokens, key_tokens, heads, kv_heads, dim, sequences
_sig("vhip_attention_workspace", _sz, _int, *_shape)
_sig("vhip_attention", _int, _int, _int, _h, _h, _h, _sz, _sz, _sz, _sz, _sz, _p, _p, _sz, _int, _f, _h, _p, _p, _sz, _p)
_sig("vhip_attention_backward_workspace", _sz, _int, *_shape)
_sig("vhip_attention_backward", _int, _int, _int, _h, _h, _h, _h, _h, _p, _sz, _sz, _sz, _sz, _sz, _p, _p, _sz, _int, _f, _h, _h,
     _h, _p, _sz, _p)


_sig("vhip_qk_norm_rotary", _int, _int, _int, _int, _h, _h, _sz, _sz, _sz, _sz, _p, _p, _p, _p, _sz, _int, _f, _h, _h, _p)
_sig("vhip_qk_norm_rotary_backward_workspace", _sz, _sz, _sz)
_sig("vhip_qk_norm_rotary_backward", _int, _int, _int, _int, _h, _h, _h, _h, _sz, _sz, _sz, _sz, _p, _p, _p, _p, _sz, _int,
     _f, _h, _h, _p, _p, _p, _sz, _p)
_sig("vhip_clip_gradients_workspace", _sz, _sz)
_sig("vhip_gradient_norm", _int, _int, _p, _sz, _p, _p, _sz, _p)
_sig("vhip_clip_gradients", _int, _int, _p, _sz, _f, _f, _p, _p, _sz, _p)


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
        # counts arrays as changed, so that a graph that saved one raises where its gradient would come of other values
        self.changed = lib.autograd.graph.increment_version if hasattr(lib, "autograd") else lambda arrays: None
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


def _heads(name, a, like=None) -> _Heads:
    """Checks rows of heads [tokens, heads, dim]."""
    if not getattr(a, "is_cuda", False):
        _on_gpu(name, a)
    st = a.stride()
    if len(st) != 3:
        raise InvalidConfig(f"{name} must have three dimensions: tokens, heads, dim")
    if like is not None and (a.dtype != like.dtype or a.get_device() != like.get_device()):
        raise InvalidConfig(f"{name} must have the type and the device of the other rows")
    n, h, d = a.shape
    if st[2] != 1 and d > 1:
        raise InvalidConfig(f"the values of a row of {name} must be contiguous")
    return _Heads(a.data_ptr(), st[0] if n > 1 else h * d, st[1] if h > 1 else d)


def _offsets(name, a, device, lib, count=None):
    """Checks the offsets of packed sequences; their address and the number of sequences."""
    _on_gpu(name, a)
    n = a.numel() - 1
    if n < 0 or (count is not None and n != count):
        raise InvalidConfig(f"{name} must hold one value more than there are sequences")
    return _vector(name, a, n + 1, device, lib.i64), n


def _attention_args(q, k, v, offsets, key_offsets, scale):
    hq, hk, hv = _heads("q", q), _heads("k", k, q), _heads("v", v, q)
    tokens, heads, dim = q.shape
    keys, kv_heads, d = k.shape
    if v.shape != k.shape or d != dim:
        raise InvalidConfig("k and v must have the same shape, and rows as long as those of q")
    if kv_heads == 0 or heads % kv_heads:
        raise InvalidConfig(f"{heads} heads are no multiple of {kv_heads}")
    device, lib = q.get_device(), _library[type(q.dtype)]
    at, n = _offsets("offsets", offsets, device, lib)
    kat = None if key_offsets is None else _offsets("key_offsets", key_offsets, device, lib, n)[0]
    if kat is None and keys != tokens:
        raise InvalidConfig("without key_offsets there are as many keys as queries")
    if scale is None:
        scale = dim ** -0.5 if dim else 1.0
    return hq, hk, hv, (tokens, keys, heads, kv_heads, dim), device, _code[q.dtype], lib, at, kat, n, scale


def attention(q, k, v, offsets, key_offsets=None, causal: bool = True, scale=None):
    """(out, lse) of softmax attention over packed sequences: q [tokens, heads, dim], k and v [tokens, kv_heads,
    dim], heads a multiple of kv_heads (query head h reads key head h // (heads // kv_heads)).  offsets (int64,
    sequences + 1 values that do not fall) bound the sequences; with key_offsets k and v have bounds of their own.
    With `causal` the last query of a sequence sees all its keys and each query before it one fewer.  scale is 1 / sqrt(dim)
    by default.  out has q's type and shape, lse is float32 [tokens, heads]; a row that sees no key, or is in no
    sequence, has out 0 and lse -inf."""
    hq, hk, hv, shape, device, code, lib, at, kat, n, scale = _attention_args(q, k, v, offsets, key_offsets, scale)
    _no_graph(lib, q, k, v)
    tokens, _, heads, _, dim = shape
    out, lse = q.new_empty((tokens, heads, dim)), q.new_empty((tokens, heads), dtype=lib.f32)
    need = _lib.vhip_attention_workspace(code, *shape, n)
    ws = q.new_empty(need, dtype=lib.u8) if need else None
    _check(_lib.vhip_attention(device, code, hq, hk, hv, *shape, at, kat, n, causal, scale,
                               _Heads(out.data_ptr(), heads * dim, dim), lse.data_ptr(),
                               None if ws is None else ws.data_ptr(), need, lib.stream(device)))
    return out, lse


def attention_backward(dout, q, k, v, out, lse, offsets, key_offsets=None, causal: bool = True, scale=None):
    """(dq, dk, dv), in the type of q, k and v, from the gradient of attention's out, its arguments and what it
    returned.  Heads that share a key head add up in its gradients; rows of no sequence have gradient 0."""
    hq, hk, hv, shape, device, code, lib, at, kat, n, scale = _attention_args(q, k, v, offsets, key_offsets, scale)
    hg, ho = _heads("dout", dout, q), _heads("out", out, q)
    if dout.shape != q.shape or out.shape != q.shape:
        raise InvalidConfig("dout and out must have the shape of q")
    tokens, keys, heads, kv_heads, dim = shape
    if lse.shape != (tokens, heads):
        raise InvalidConfig("lse must hold a value for each token and head")
    ls = _vector("lse", lse.view(-1) if lse.is_contiguous() else lse, tokens * heads, device, lib.f32)
    dq, dk, dv = q.new_empty((tokens, heads, dim)), k.new_empty((keys, kv_heads, dim)), k.new_empty((keys, kv_heads, dim))
    need = _lib.vhip_attention_backward_workspace(code, *shape, n)
    ws = q.new_empty(need, dtype=lib.u8)
    rows = lambda a, h: _Heads(a.data_ptr(), h * dim, dim)  # noqa: E731
    _check(_lib.vhip_attention_backward(device, code, hg, hq, hk, hv, ho, ls, *shape, at, kat, n, causal, scale,
                                        rows(dq, heads), rows(dk, kv_heads), rows(dv, kv_heads), ws.data_ptr(), need,
                                        lib.stream(device)))
    return dq, dk, dv


def _head_args(q, k, q_weight, k_weight, positions, frequencies):
    hq, hk = _heads("q", q), _heads("k", k, q)
    tokens, heads, dim = q.shape
    if k.shape[0] != tokens or k.shape[2] != dim:
        raise InvalidConfig("q and k must have the same tokens, and rows of the same length")
    device, code, lib = q.get_device(), _code[q.dtype], _library[type(q.dtype)]
    wq = wk = None
    params = code
    if (q_weight is None) != (k_weight is None):
        raise InvalidConfig("q_weight and k_weight are given together or not at all")
    if q_weight is not None:
        wq, wk = _vector("q_weight", q_weight, dim, device), _vector("k_weight", k_weight, dim, device)
        if q_weight.dtype != k_weight.dtype:
            raise InvalidConfig("q_weight and k_weight must have the same type")
        params = _param_code(q_weight.dtype, code)
    at = _vector("positions", positions, tokens, device, lib.i64)
    _on_gpu("frequencies", frequencies)
    pairs = frequencies.numel()
    fr = _vector("frequencies", frequencies, pairs, device, lib.f32)
    return hq, hk, (tokens, heads, k.shape[1], dim), device, code, params, lib, wq, wk, at, fr, 2 * pairs


def qk_norm_rotary(q, k, q_weight, k_weight, positions, frequencies, eps: float = 1e-6, interleaved: bool = False):
    """(q', k') of queries [tokens, heads, dim] and keys [tokens, kv_heads, dim]: each row over its root mean square,
    x / sqrt(mean x^2 + eps), times the weight (dim values; both None: 1), its first 2 len(frequencies) columns
    turned by their token's position (int64): pair i by positions[t] * frequencies[i] radians (float32, their product in
    64 bits).  Pairs are columns i and i + len(frequencies), or with `interleaved` 2 i and 2 i + 1."""
    hq, hk, shape, device, code, params, lib, wq, wk, at, fr, rotary = _head_args(q, k, q_weight, k_weight, positions, frequencies)
    _no_graph(lib, q, k, q_weight, k_weight, frequencies)
    tokens, heads, kv_heads, dim = shape
    qo, ko = q.new_empty((tokens, heads, dim)), k.new_empty((tokens, kv_heads, dim))
    _check(_lib.vhip_qk_norm_rotary(device, code, params, hq, hk, *shape, wq, wk, at, fr, rotary, interleaved, eps,
                                    _Heads(qo.data_ptr(), heads * dim, dim), _Heads(ko.data_ptr(), kv_heads * dim, dim),
                                    lib.stream(device)))
    return qo, ko


def qk_norm_rotary_backward(dq, dk, q, k, q_weight, k_weight, positions, frequencies, eps: float = 1e-6,
                            interleaved: bool = False):
    """(dq, dk, dq_weight, dk_weight) from the gradients of qk_norm_rotary's outputs and its arguments.  The weights'
    gradients have their type; without weights they are None."""
    hq, hk, shape, device, code, params, lib, wq, wk, at, fr, rotary = _head_args(q, k, q_weight, k_weight, positions, frequencies)
    gq, gk = _heads("dq", dq, q), _heads("dk", dk, q)
    if dq.shape != q.shape or dk.shape != k.shape:
        raise InvalidConfig("dq and dk must have the shapes of q and k")
    tokens, heads, kv_heads, dim = shape
    qo, ko = q.new_empty((tokens, heads, dim)), k.new_empty((tokens, kv_heads, dim))
    dqw = dkw = ws = None
    need = 0
    if wq is not None:
        dqw, dkw = q_weight.new_empty((2, dim)).unbind()
        need = _lib.vhip_qk_norm_rotary_backward_workspace(tokens, dim)
        ws = q.new_empty(need, dtype=lib.u8)
    at_of = lambda a: None if a is None else a.data_ptr()  # noqa: E731
    _check(_lib.vhip_qk_norm_rotary_backward(device, code, params, gq, gk, hq, hk, *shape, wq, wk, at, fr, rotary, interleaved,
                                             eps, _Heads(qo.data_ptr(), heads * dim, dim),
                                             _Heads(ko.data_ptr(), kv_heads * dim, dim), at_of(dqw), at_of(dkw), at_of(ws),
                                             need, lib.stream(device)))
    return qo, ko, dqw, dkw


def _dense(a) -> bool:
    """Whether an array's values fill a block of memory, in whatever order of its dimensions."""
    if a.is_contiguous():
        return True
    size = 1
    for stride, n in sorted((st, n) for st, n in zip(a.stride(), a.shape) if n != 1):
        if stride != size:
            return False
        size *= n
    return True


def _arrays(gradients, out):
    if not gradients:
        raise InvalidConfig("there is no array")
    first = gradients[0]
    _on_gpu("a gradient", first)
    device, lib = first.get_device(), _library[type(first.dtype)]
    table = array("Q")  # of vhip_array: data, out, count, and the two types in one
    # the other arrays are of the first one's kind: an array in host memory has no device number, or -1
    try:
        if out is None:
            for g in gradients:
                if g.get_device() != device:
                    raise InvalidConfig("the gradients are not all on one GPU")
                if not (g.is_contiguous() or _dense(g)):
                    raise InvalidConfig("the values of a gradient must fill a block of memory")
                at, code = g.data_ptr(), _code[g.dtype]
                table.extend((at, at, g.numel(), code | code << 32))
        else:
            if len(out) != len(gradients):
                raise InvalidConfig("out must hold an array for each gradient")
            for g, o in zip(gradients, out):
                if not g.get_device() == o.get_device() == device:
                    raise InvalidConfig("the gradients and the outputs are not all on one GPU")
                if o.shape != g.shape:
                    raise InvalidConfig("an output must have the shape of its gradient")
                if not (g.is_contiguous() and o.is_contiguous()) and not (_dense(g) and g.stride() == o.stride()):
                    raise InvalidConfig("a gradient and its output must fill blocks of memory in the same order")
                table.extend((g.data_ptr(), o.data_ptr(), g.numel(), _code[g.dtype] | _code[o.dtype] << 32))
    except AttributeError:
        raise InvalidConfig("the gradients and the outputs are not all arrays in GPU memory") from None
    need = _lib.vhip_clip_gradients_workspace(len(gradients))
    return table, len(gradients), first.new_empty((), dtype=lib.f32), first.new_empty(need, dtype=lib.u8), need, device, lib


def gradient_norm(gradients):
    """The norm (float32, no dimensions) of all values of a list of arrays together: sqrt(sum g^2), in 64 bits until it
    is rounded.  The arrays are of any of the types, each filling a block of memory."""
    gradients = list(gradients)
    table, n, norm, ws, need, device, lib = _arrays(gradients, None)
    _no_graph(lib, *gradients)
    _check(_lib.vhip_gradient_norm(device, table.buffer_info()[0], n, norm.data_ptr(), ws.data_ptr(), need, lib.stream(device)))
    return norm


def clip_gradients(gradients, max_norm: float, out=None, eps: float = 1e-6):
    """gradient_norm of the arrays; each is scaled by min(1, max_norm / (norm + eps)), in place or into the arrays `out`
    (the same shapes, any of the types), which overlap nothing else.  A norm that is infinite or NaN is no error: it
    leaves zeros and NaN.  What is written counts as changed: a graph of torch that saved it raises."""
    gradients = list(gradients)
    out = None if out is None else list(out)
    table, n, norm, ws, need, device, lib = _arrays(gradients, out)
    _no_graph(lib, *gradients, *(out or ()))
    _check(_lib.vhip_clip_gradients(device, table.buffer_info()[0], n, max_norm, eps, norm.data_ptr(), ws.data_ptr(), need, lib.stream(device)))
    lib.changed(gradients if out is None else out)
    return norm
