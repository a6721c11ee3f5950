"""Argument checks of attention, head norms and clipping at the C ABI, on the CPU: every refusal comes before a device
is used."""
import ctypes
import math

import pytest

BAD = -5  # VHIP_ERR_INVALID_CONFIG
F32, F16, BF16 = 0, 1, 2
P = 4096  # a pointer that no call gets to use
NAN, INF = math.nan, math.inf


@pytest.fixture(scope="module")
def tr():
    from vector_hip import training  # declares the signatures

    return training


def heads(tr, data=P, token=64, head=32):
    return tr._Heads(data, token, head)


def call(name, tr, values, wrong):
    a = dict(values)
    for k, v in wrong.items():
        assert k in a, k
        a[k] = heads(tr, **v) if isinstance(v, dict) else v
    return getattr(tr._lib, name)(*a.values())


SHAPE = dict(tokens=6, key_tokens=6, heads=2, kv_heads=2, dim=32)


def attn(tr, **wrong):
    return call("vhip_attention", tr, dict(ordinal=0, dtype=F32, q=heads(tr), k=heads(tr), v=heads(tr), **SHAPE, offsets=P,
                key_offsets=None, sequences=1, causal=1, scale=1.0, out=heads(tr), lse=P, ws=P, bytes=1 << 30, stream=None), wrong)


def attn_back(tr, **wrong):
    return call("vhip_attention_backward", tr, dict(ordinal=0, dtype=F32, dout=heads(tr), q=heads(tr), k=heads(tr), v=heads(tr),
                out=heads(tr), lse=P, **SHAPE, offsets=P, key_offsets=None, sequences=1, causal=1, scale=1.0, dq=heads(tr),
                dk=heads(tr), dv=heads(tr), ws=P, bytes=1 << 30, stream=None), wrong)


def norm(tr, **wrong):
    return call("vhip_qk_norm_rotary", tr, dict(ordinal=0, dtype=F32, param=F32, q=heads(tr), k=heads(tr), tokens=6, heads=2, kv_heads=2,
                dim=32, qw=P, kw=P, positions=P, frequencies=P, rotary=32, near=0, eps=1e-6, qo=heads(tr), ko=heads(tr),
                stream=None), wrong)


def norm_back(tr, **wrong):
    return call("vhip_qk_norm_rotary_backward", tr, dict(ordinal=0, dtype=F32, param=F32, dq=heads(tr), dk=heads(tr), q=heads(tr),
                k=heads(tr), tokens=6, heads=2, kv_heads=2, dim=32, qw=P, kw=P, positions=P, frequencies=P, rotary=32, near=0, eps=1e-6,
                dqo=heads(tr), dko=heads(tr), dqw=P, dkw=P, ws=P, bytes=1 << 20, stream=None), wrong)


class Array(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("out", ctypes.c_void_p), ("count", ctypes.c_size_t), ("dtype", ctypes.c_int), ("out_dtype", ctypes.c_int)]


def clip(tr, rows=((P, P, 10, F32, F32),), count=None, **wrong):
    table = (Array * max(1, len(rows)))(*rows)
    return call("vhip_clip_gradients", tr, dict(ordinal=0, arrays=ctypes.addressof(table), count=len(rows) if count is None else count,
                max_norm=1.0, eps=1e-6, norm=P, ws=P, bytes=1 << 20, stream=None), wrong)


@pytest.mark.parametrize("what,wrong", [
    (attn, dict(dtype=3)), (attn, dict(dtype=-1)), (attn, dict(dim=0)), (attn, dict(dim=129, q=dict(token=258, head=129))), (attn, dict(heads=0)),
    (attn, dict(kv_heads=0)), (attn, dict(heads=3)), (attn, dict(offsets=None)), (attn, dict(key_tokens=7)), (attn, dict(scale=NAN)),
    (attn, dict(scale=INF)), (attn, dict(scale=-1e31)), (attn, dict(q=dict(data=None))), (attn, dict(k=dict(data=None))), (attn, dict(v=dict(data=None))), (attn, dict(out=dict(data=None))),
    (attn, dict(q=None)), (attn, dict(q=dict(token=31))), (attn, dict(k=dict(token=63))), (attn, dict(v=dict(head=31))), (attn, dict(out=dict(token=33, head=32))),
    (attn, dict(q=dict(data=P + 2))), (attn, dict(k=dict(token=(1 << 23) + 1))), (attn, dict(v=dict(token=32, head=(1 << 40) + 1))), (attn, dict(tokens=1 << 31)),
    (attn, dict(tokens=1 << 30, key_tokens=1 << 30)), (attn, dict(sequences=1 << 29)), (attn, dict(key_offsets=P, key_tokens=100_000, ws=None)),
    (attn, dict(key_offsets=P, key_tokens=100_000, bytes=64)), (attn, dict(key_offsets=P, key_tokens=100_000, ws=P + 8)),
    (attn_back, dict(dtype=9)), (attn_back, dict(lse=None)), (attn_back, dict(dout=dict(data=None))), (attn_back, dict(out=dict(data=None))),
    (attn_back, dict(dq=dict(data=None))), (attn_back, dict(dk=dict(token=63))), (attn_back, dict(dv=None)), (attn_back, dict(ws=None)), (attn_back, dict(bytes=16)),
    (attn_back, dict(ws=P + 4)), (attn_back, dict(heads=5)), (attn_back, dict(scale=NAN)),
    (norm, dict(dtype=7)), (norm, dict(param=F16)), (norm, dict(dim=0)), (norm, dict(dim=257, q=dict(token=600, head=300))), (norm, dict(rotary=34)), (norm, dict(rotary=3)),
    (norm, dict(heads=0, kv_heads=0)), (norm, dict(tokens=1 << 31)), (norm, dict(positions=None)), (norm, dict(frequencies=None)), (norm, dict(eps=-1.0)),
    (norm, dict(eps=NAN)), (norm, dict(q=dict(data=None))), (norm, dict(ko=dict(token=63))), (norm, dict(qo=None)), (norm, dict(k=dict(data=P + 1))),
    (norm_back, dict(dq=dict(data=None))), (norm_back, dict(dko=dict(head=31))), (norm_back, dict(ws=None)), (norm_back, dict(bytes=255)), (norm_back, dict(ws=P + 2)),
    (clip, dict(max_norm=-1.0)), (clip, dict(max_norm=NAN)), (clip, dict(eps=-1.0)), (clip, dict(eps=NAN)), (clip, dict(ws=None)), (clip, dict(bytes=100)), (clip, dict(ws=P + 4)),
    (clip, dict(arrays=None)), (clip, dict(rows=((P, P, 10, 5, F32),))), (clip, dict(rows=((P, P + 100, 10, F32, 5),))), (clip, dict(rows=((None, P, 10, F32, F32),))),
    (clip, dict(rows=((P, None, 10, F32, F32),))), (clip, dict(rows=((P + 2, P + 2, 10, F32, F32),))), (clip, dict(rows=((P, P, 10, F32, F16),))),
    (clip, dict(rows=((P, P, 1 << 41, F32, F32),))), (clip, dict(rows=((P, P, 10, F32, F32), (P, P, 10, F32, F32)))),
    (clip, dict(rows=((P, 2 * P, 10, F32, F32), (2 * P + 36, 3 * P, 10, F32, F32)))), (clip, dict(rows=((P, 2 * P, 10, F32, F32), (3 * P, 2 * P + 20, 10, F32, BF16)))),
    (clip, dict(rows=((P, P + 4, 10, F32, F32), (2 * P, 2 * P, 1, F32, F32)))),
    (clip, dict(rows=((P, P, 1000, F32, F32), (P + 8, 3 * P, 10, F32, F32)))),
])
def test_refused(tr, what, wrong):
    assert what(tr, **wrong) == BAD
    assert tr._lib.vhip_last_error()


@pytest.mark.parametrize("what,right", [
    (attn, dict()), (attn, dict(q=dict(token=32, head=192))), (attn, dict(tokens=1, key_tokens=1, q=dict(token=0))), (attn, dict(dtype=BF16, key_offsets=P, key_tokens=0)),
    (attn, dict(tokens=0, key_tokens=0, q=dict(data=None))), (attn_back, dict()), (attn_back, dict(key_offsets=P, key_tokens=0)), (norm, dict()), (norm, dict(rotary=0, positions=None, frequencies=None)),
    (norm, dict(kv_heads=0, k=dict(data=None))), (norm_back, dict(dqw=None, dkw=None, ws=None)), (clip, dict()), (clip, dict(rows=())),
    (clip, dict(rows=((P, P, 10, F32, F32), (P + 40, P + 40, 10, F32, F32)))), (clip, dict(rows=((P, 2 * P, 10, BF16, F32), (P, 3 * P, 10, BF16, BF16)))),
    (clip, dict(rows=((None, None, 0, F32, F32), (P, P, 3, F16, F16)))), (clip, dict(max_norm=INF)), (clip, dict(norm=None)),
])
def test_not_refused(tr, what, right):
    """All checks are passed: the call gets as far as looking for its GPU."""
    missing = tr._lib.vhip_device_count() + 100
    assert what(tr, ordinal=missing, **right) not in (0, BAD)


def test_workspaces(tr):
    lib = tr._lib
    one, many = (BF16, 1, 100_000, 8, 2, 128, 1), (BF16, 100_000, 100_000, 8, 2, 128, 10)
    assert lib.vhip_attention_workspace(*one) > 0 and lib.vhip_attention_workspace(*many) == 0
    assert lib.vhip_attention_backward_workspace(*many) >= 4 * 100_000 * 8
    # parts are bounded: their sums are no more than a quarter of what is read, or 64 of few rows
    assert lib.vhip_attention_workspace(*one) <= 64 * 8 * (128 * 4 + 8)
    for sizes in ((0, 0, 1, 1, 1, 0), (0, 5, 2, 1, 64, 3), (5, 0, 2, 1, 64, 3), (1, 1, 1, 1, 1, 0)):
        lib.vhip_attention_workspace(F32, *sizes)
        lib.vhip_attention_backward_workspace(F32, *sizes)
    assert lib.vhip_attention_workspace(F32, 1, 1, 1, 0, 1, 1) == lib.vhip_attention_backward_workspace(F32, 1, 1, 0, 1, 1, 1) == 0
    assert lib.vhip_qk_norm_rotary_backward_workspace(0, 64) == 0
    assert lib.vhip_qk_norm_rotary_backward_workspace(1 << 20, 64) == 2 * 4 * 64 * 1024
    assert lib.vhip_clip_gradients_workspace(1) <= lib.vhip_clip_gradients_workspace(1000) <= 8 * 4096


def test_arrays_on_the_host_are_refused(tr):
    import numpy as np

    import vector_hip as vh

    class Host(np.ndarray):
        is_cuda = False

    for x in (np.zeros((4, 2, 8), np.float32), np.zeros((4, 2, 8), np.float32).view(Host), [1.0], None):
        for f in (lambda: tr.attention(x, x, x, x), lambda: tr.attention_backward(x, x, x, x, x, x, x), lambda: tr.qk_norm_rotary(x, x, None, None, x, x),
                  lambda: tr.qk_norm_rotary_backward(x, x, x, x, None, None, x, x), lambda: tr.gradient_norm([x]), lambda: tr.clip_gradients([x], 1.0)):
            with pytest.raises(vh.InvalidConfig):
                f()
    for nothing in (tr.gradient_norm, lambda a: tr.clip_gradients(a, 1.0)):
        with pytest.raises(vh.InvalidConfig):
            nothing([])
