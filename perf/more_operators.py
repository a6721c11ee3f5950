"""The operators of an encoder's attention and of its training step, as cases that can be timed and compared.

Three operators lie between a model's tokens and the head of ``operators.py``:

* ``qk``         the queries' and keys' norm for each head with the rotation by their positions in the same pass:
                 ``forward`` gives both, ``backward`` their gradients and those of the two weights;
* ``attention``  softmax attention of packed sequences of different lengths with grouped heads, causal or not:
                 ``forward`` gives the output and the log-sum-exp of each row, ``grad`` these and the gradients of
                 queries, keys and values;
* ``clip``       the norm of a model's gradients over all its arrays, and their clipped values.

``listed()`` holds the sizes at which these are used; ``draw()`` gives others of the same ranges.  ``run`` computes a
case in plain torch operations in 32 bits, or, where ``own`` is true, by the package's own calls.
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vector-rs_amd"))

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
QK_EPS = 1e-6
CLIP_EPS = 1e-6


def listed():
    return [
        # one token of a request: latency alone
        {"name": "qk_fwd_1x12x12x64_f32", "op": "qk", "pass": "forward", "tokens": 1, "heads": 12, "kv_heads": 12,
         "dim": 64, "rotary": 64, "interleaved": False, "dtype": "f32", "params": "f32", "packed": False, "far": 512},
        # a batch of long prompts, queries and keys as the projection's output holds them
        {"name": "qk_fwd_16384x32x8x128_bf16", "op": "qk", "pass": "forward", "tokens": 16384, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "dtype": "bf16", "params": "bf16",
         "packed": True, "far": 32768},
        # a training batch: odd count of tokens, half of each head rotated in neighbouring pairs, far positions
        {"name": "qk_bwd_8191x16x4x80_f16", "op": "qk", "pass": "backward", "tokens": 8191, "heads": 16, "kv_heads": 4,
         "dim": 80, "rotary": 40, "interleaved": True, "dtype": "f16", "params": "f32", "packed": True,
         "far": 1_000_000},
        # one query text through an encoder in full precision: latency alone
        {"name": "attn_fwd_1x19_12x12x64_f32", "op": "attention", "pass": "forward", "sequences": 1, "shortest": 19,
         "longest": 19, "earlier": 0, "deal": 1, "heads": 12, "kv_heads": 12, "dim": 64, "causal": False,
         "dtype": "f32"},
        # indexing: texts of 16 to 512 tokens through an encoder that looks both ways
        {"name": "attn_fwd_256x16-512_12x12x64_bf16", "op": "attention", "pass": "forward", "sequences": 256,
         "shortest": 16, "longest": 512, "earlier": 0, "deal": 2, "heads": 12, "kv_heads": 12, "dim": 64,
         "causal": False, "dtype": "bf16"},
        # the last token of each of a few long texts against all that came before: one pass over the keys and values
        {"name": "attn_fwd_5x1+65536_32x8x128_bf16", "op": "attention", "pass": "forward", "sequences": 5,
         "shortest": 1, "longest": 1, "earlier": 65536, "deal": 3, "heads": 32, "kv_heads": 8, "dim": 128,
         "causal": True, "dtype": "bf16"},
        # a whole long document, causal with grouped heads: the largest
        {"name": "attn_fwd_1x32768_32x8x128_bf16", "op": "attention", "pass": "forward", "sequences": 1,
         "shortest": 32768, "longest": 32768, "earlier": 0, "deal": 4, "heads": 32, "kv_heads": 8, "dim": 128,
         "causal": True, "dtype": "bf16"},
        # a small training step over short texts, heads whose size is no power of two
        {"name": "attn_grad_9x1-200_6x2x72_f16", "op": "attention", "pass": "grad", "sequences": 9, "shortest": 1,
         "longest": 200, "earlier": 0, "deal": 5, "heads": 6, "kv_heads": 2, "dim": 72, "causal": True,
         "dtype": "f16"},
        # a training step over packed documents of ragged lengths
        {"name": "attn_grad_8x512-8192_16x4x128_bf16", "op": "attention", "pass": "grad", "sequences": 8,
         "shortest": 512, "longest": 8192, "earlier": 0, "deal": 6, "heads": 16, "kv_heads": 4, "dim": 128,
         "causal": True, "dtype": "bf16"},
        # the arrays of a retriever with a small table: latency alone
        {"name": "clip_0x64+1000_f32", "op": "clip", "layers": 0, "dim": 64, "table": 1000, "dtype": "f32",
         "out": "f32", "flat": False, "limit": 1.0},
        # arrays of odd sizes one after the other in a communication buffer, under mixed precision
        {"name": "clip_6x333+30000_f16", "op": "clip", "layers": 6, "dim": 333, "table": 30_000, "dtype": "f16",
         "out": "f32", "flat": True, "limit": 1.0},
        # all of an encoder with a large table
        {"name": "clip_9x1536+131072_bf16", "op": "clip", "layers": 9, "dim": 1536, "table": 131_072,
         "dtype": "bf16", "out": "bf16", "flat": False, "limit": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk", "attention", "attention", "clip"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "clip":
        return {"op": op, "layers": rng.randint(0, 9), "dim": _log(rng, 16, 1536), "table": _log(rng, 1000, 131_072),
                "dtype": dtype, "out": rng.choice([dtype, "f32"]), "flat": rng.random() < 0.5,
                "limit": rng.choice([0.1, 1.0, 1000.0])}
    kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4])
    dim = _log(rng, 16, 128)
    dim = rng.choice([64, 128, (dim + 7) // 8 * 8, (dim + 1) // 2 * 2])
    case = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    if op == "qk":
        return dict(case, tokens=_log(rng, 1, 16384), rotary=rng.choice([dim, dim // 4 * 2]),
                    interleaved=rng.random() < 0.5, params=rng.choice([dtype, "f32"]), packed=rng.random() < 0.5,
                    far=rng.choice([512, 32768, 1_000_000]), **{"pass": rng.choice(["forward", "backward"])})
    longest = _log(rng, 1, 16384)
    case.update(sequences=_log(rng, 1, 64), shortest=_log(rng, 1, longest), longest=longest,
                earlier=rng.choice([0, 0, _log(rng, 1, 65536)]), deal=rng.randrange(1 << 30),
                causal=rng.random() < 0.6, **{"pass": rng.choice(["forward", "grad"])})
    # no more than a tenth of the largest case's work, and in 32 bits, where each costs more, a hundredth
    limit = 8.8e12 / (100 if dtype == "f32" else 10)
    while work(case)["flops"] > limit or sum(_lengths(case)[1]) * case["heads"] * dim > 1 << 28:
        if case["sequences"] > 1:
            case["sequences"] = (case["sequences"] + 1) // 2
        else:
            case["longest"] = (case["longest"] + 1) // 2
            case["shortest"] = min(case["shortest"], case["longest"])
            case["earlier"] //= 2
    return case


def _lengths(case):
    """Queries and keys of each sequence: those of its own, and keys that came before them."""
    rng = random.Random(case["deal"])
    lq = [_log(rng, case["shortest"], case["longest"]) for _ in range(case["sequences"])]
    before = [_log(rng, (case["earlier"] + 15) // 16, case["earlier"]) if case["earlier"] else 0 for _ in lq]
    return lq, [n + b for n, b in zip(lq, before)]


def _shapes(case):
    d = case["dim"]
    layer = [(d,), (3 * d, d), (d, d), (d,), (4 * d, d), (d, 4 * d)]
    return [(case["table"], d)] + layer * case["layers"] + [(d,), (d, d)]


def work(case):
    s = BYTES[case["dtype"]]
    if case["op"] == "clip":
        n = sum(math.prod(shape) for shape in _shapes(case))
        return {"bytes": n * (s + BYTES[case["out"]]), "flops": 3 * n}
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "qk":
        n = case["tokens"] * (h + g) * d
        extra = 8 * case["tokens"] + 2 * case["rotary"]
        if case["pass"] == "forward":
            return {"bytes": 2 * n * s + extra + 2 * d * BYTES[case["params"]], "flops": 7 * n}
        return {"bytes": 3 * n * s + extra + 4 * d * BYTES[case["params"]], "flops": 13 * n}
    lq, lk = _lengths(case)
    pairs = sum(q * (k - q) + q * (q + 1) // 2 if case["causal"] else q * k for q, k in zip(lq, lk))
    tq, tk = sum(lq) * h, sum(lk) * g
    forward = 2 * (tq + tk) * d * s + 4 * tq
    if case["pass"] == "forward":
        return {"bytes": forward, "flops": 4 * pairs * h * d}
    return {"bytes": forward + (2 * tq + 2 * tk) * d * s, "flops": 14 * pairs * h * d}


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    if case["op"] == "clip":
        shapes = _shapes(case)
        sizes = [math.prod(shape) for shape in shapes]
        if case["flat"]:  # views of one buffer, as a communication bucket holds them
            ends = _offsets(sizes)
            flat = torch.empty(ends[-1], device="cuda", dtype=dtype)
            outs = torch.empty(ends[-1], device="cuda", dtype=TYPES[case["out"]])
            grads = [flat[b:e].view(shape) for b, e, shape in zip(ends, ends[1:], shapes)]
            out = [outs[b:e].view(shape) for b, e, shape in zip(ends, ends[1:], shapes)]
        else:
            grads = [torch.empty(shape, device="cuda", dtype=dtype) for shape in shapes]
            out = [torch.empty(shape, device="cuda", dtype=TYPES[case["out"]]) for shape in shapes]
        for i, g in enumerate(grads):  # later layers have larger gradients
            g.copy_(normal(*g.shape).mul_(1e-2 * (1 + i) / len(grads)))
        return {"case": case, "gradients": grads, "out": out}
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "qk":
        n, params = case["tokens"], TYPES[case["params"]]
        # channels of different widths, some far larger, as trained projections give them
        width = torch.exp(0.7 * normal(h + 2 * g, d))
        if case["packed"]:
            qkv = (normal(n, h + 2 * g, d) * width).to(dtype)
            q, k = qkv[:, :h], qkv[:, h:h + g]
        else:
            q, k = (normal(n, h, d) * width[:h]).to(dtype), (normal(n, g, d) * width[:g]).to(dtype)
        rot = case["rotary"]
        state = {"q": q, "k": k, "q_weight": (1 + 0.2 * normal(d)).to(params),
                 "k_weight": (1 + 0.2 * normal(d)).to(params),
                 "positions": torch.randint(0, case["far"], (n,), device="cuda", generator=gen),
                 "frequencies": 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float32) / max(rot, 1))}
        if case["pass"] == "backward":
            state.update(dq=(0.01 * normal(n, h, d)).to(dtype), dk=(0.01 * normal(n, g, d)).to(dtype))
        return dict(state, case=case)
    lq, lk = _lengths(case)
    tq, tk = sum(lq), sum(lk)
    # queries and keys after their norm; a few channels weigh more, so that rows attend to some keys far more
    weight = torch.exp(0.4 * normal(d))
    state = {"q": (normal(tq, h, d) * weight).to(dtype), "k": (normal(tk, g, d) * weight).to(dtype)}
    if case["earlier"]:
        state["v"] = normal(tk, g, d).to(dtype)
    else:  # values are read where the projection of all three left them
        state["v"] = normal(tk, h + 2 * g, d).to(dtype)[:, h + g:]
    state["offsets"] = torch.tensor(_offsets(lq), device="cuda", dtype=torch.int64)
    state["key_offsets"] = torch.tensor(_offsets(lk), device="cuda", dtype=torch.int64) if case["earlier"] else None
    if case["pass"] == "grad":
        state["dout"] = (0.01 * normal(tq, h, d)).to(dtype)
    return dict(state, case=case, lengths=(lq, lk))


# ---- plain forms, in 32 bits -------------------------------------------------------------------------------------


def _clip(s):
    total = torch.zeros((), device="cuda", dtype=torch.float64)
    for g in s["gradients"]:
        g = g.float()
        total += (g * g).sum(dtype=torch.float64)
    norm = total.sqrt()
    c = (s["case"]["limit"] / (norm + CLIP_EPS)).clamp(max=1.0).float()
    for g, o in zip(s["gradients"], s["out"]):
        o.copy_(g.float() * c)
    return {"norm": norm.float(), "out": s["out"]}


def _rotation(s):
    angle = s["positions"].double()[:, None] * s["frequencies"].double()
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _halves(x, rot, interleaved):
    if interleaved:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def _rotated(x, cos, sin, rot, interleaved):
    a, b = _halves(x, rot, interleaved)
    out = x.clone()
    oa, ob = _halves(out, rot, interleaved)
    oa.copy_(a * cos - b * sin)
    ob.copy_(a * sin + b * cos)
    return out


def _qk(s):
    case = s["case"]
    rot, il = case["rotary"], case["interleaved"]
    cos, sin = _rotation(s)
    out = {}
    for name in "qk":
        x, w = s[name].float(), s[name + "_weight"].float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + QK_EPS)
        if case["pass"] == "forward":
            out[name] = _rotated(x * r * w, cos, sin, rot, il).to(s[name].dtype)
            continue
        dn = _rotated(s["d" + name].float(), cos, -sin, rot, il)
        xh, u = x * r, dn * w
        out["d" + name] = (r * (u - xh * (u * xh).mean(-1, keepdim=True))).to(s[name].dtype)
        out["d" + name + "_weight"] = (dn * xh).sum((0, 1)).to(s[name + "_weight"].dtype)
    return out


def _attention(s):
    case = s["case"]
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    grad, scale, per = case["pass"] == "grad", 1 / math.sqrt(d), h // g
    q, k, v = s["q"], s["k"], s["v"]
    out, lse = torch.empty_like(q), torch.empty(q.shape[0], h, device="cuda")
    if grad:
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty(v.shape, device="cuda", dtype=v.dtype)
    qb = kb = 0
    for lq, lk in zip(*s["lengths"]):
        ks, vs = (x[kb:kb + lk].float().transpose(0, 1).contiguous() for x in (k, v))  # [kv_heads, lk, d]
        kt, vt = ks.transpose(1, 2).contiguous(), vs.transpose(1, 2).contiguous()
        if grad:
            sk, sv = torch.zeros_like(ks), torch.zeros_like(vs)
        step = max(1, min(lq, (1 << 29) // (h * lk)))
        for b in range(0, lq, step):
            e = min(lq, b + step)
            # rows of a group beside one another: [kv_heads, rows * per, d]
            fold = lambda x: x[qb + b:qb + e].float().view(e - b, g, per * d).transpose(0, 1).reshape(g, (e - b) * per, d)  # noqa: E731,B023
            unfold = lambda x: x.view(g, e - b, per, -1).transpose(0, 1).reshape(e - b, h, -1)  # noqa: E731,B023
            qs = fold(q)
            z = torch.bmm(qs, kt) * scale
            if case["causal"]:
                i = torch.arange(b, e, device="cuda").repeat_interleave(per)[:, None]
                z.masked_fill_(torch.arange(lk, device="cuda") > i + (lk - lq), -math.inf)
            top = z.max(2, keepdim=True).values
            z = torch.exp(z.sub_(top))
            total = z.sum(2, keepdim=True)
            o = torch.bmm(z, vs) / total
            out[qb + b:qb + e] = unfold(o).to(out.dtype)
            lse[qb + b:qb + e] = unfold(top + torch.log(total))[:, :, 0]
            if grad:
                do, p = fold(s["dout"]), z.div_(total)
                sv += torch.bmm(p.transpose(1, 2).contiguous(), do)
                dz = torch.bmm(do, vt).sub_((do * o).sum(2, keepdim=True)).mul_(p).mul_(scale)
                dq[qb + b:qb + e] = unfold(torch.bmm(dz, ks)).to(dq.dtype)
                sk += torch.bmm(dz.transpose(1, 2).contiguous(), qs)
        if grad:
            dk[kb:kb + lk], dv[kb:kb + lk] = sk.transpose(0, 1).to(dk.dtype), sv.transpose(0, 1).to(dv.dtype)
        qb, kb = qb + lq, kb + lk
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv} if grad else {"out": out, "lse": lse}


def _own(s):
    from vector_hip import training

    case = s["case"]
    if case["op"] == "clip":
        norm = training.clip_gradients(s["gradients"], case["limit"], out=s["out"], eps=CLIP_EPS)
        return {"norm": norm, "out": s["out"]}
    if case["op"] == "qk":
        how = {"eps": QK_EPS, "interleaved": case["interleaved"]}
        at = (s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["frequencies"])
        if case["pass"] == "forward":
            return dict(zip("qk", training.qk_norm_rotary(*at, **how)))
        return dict(zip(("dq", "dk", "dq_weight", "dk_weight"),
                        training.qk_norm_rotary_backward(s["dq"], s["dk"], *at, **how)))
    packed = {"key_offsets": s["key_offsets"], "causal": case["causal"]}
    q, k, v = s["q"], s["k"], s["v"]
    out, lse = training.attention(q, k, v, s["offsets"], **packed)
    if case["pass"] == "forward":
        return {"out": out, "lse": lse}
    dq, dk, dv = training.attention_backward(s["dout"], q, k, v, out, lse, s["offsets"], **packed)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def run(state):
    if own:
        return _own(state)
    return {"clip": _clip, "qk": _qk, "attention": _attention}[state["case"]["op"]](state)


# ---- the definitions, in 64 bits ---------------------------------------------------------------------------------


def _exact_clip(s):
    norm = torch.stack([torch.linalg.vector_norm(g.double()) for g in s["gradients"]]).norm()
    c = min(1.0, s["case"]["limit"] / (float(norm) + CLIP_EPS))
    return {"norm": norm, "out": [g.double() * c for g in s["gradients"]]}


def _exact_head_norm(x, weight, positions, frequencies, interleaved):
    """A rotation as a product with a complex number of length one."""
    x = x / (x.square().mean(-1, keepdim=True) + QK_EPS).sqrt() * weight
    rot = 2 * len(frequencies)
    turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64),
                       positions.double()[:, None] * frequencies.double())[:, None]
    first = x[..., :rot].unflatten(-1, (-1, 2) if interleaved else (2, -1))
    axis = -1 if interleaved else -2
    z = torch.complex(*first.unbind(axis)) * turn
    first = torch.stack((z.real, z.imag), axis).flatten(-2)
    return torch.cat((first, x[..., rot:]), -1)


def _exact_qk(s):
    case, out = s["case"], {}
    for name in "qk":
        x = s[name].double().contiguous().requires_grad_()
        w = s[name + "_weight"].double().requires_grad_()
        with torch.enable_grad():
            y = _exact_head_norm(x, w, s["positions"], s["frequencies"], case["interleaved"])
            if case["pass"] == "forward":
                out[name] = y.detach()
            else:
                out["d" + name], out["d" + name + "_weight"] = torch.autograd.grad(y, (x, w), s["d" + name].double())
    return out


def _exact_attention(s):
    """Head by head, gradients by automatic differentiation."""
    case = s["case"]
    h, per, d = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
    grad = case["pass"] == "grad"
    new = lambda x: torch.zeros(x.shape, device="cuda", dtype=torch.float64)  # noqa: E731
    out = {"out": new(s["q"]), "lse": torch.zeros(s["q"].shape[0], h, device="cuda", dtype=torch.float64)}
    if grad:
        out.update(dq=new(s["q"]), dk=new(s["k"]), dv=new(s["v"]))
    qb = kb = 0
    for lq, lk in zip(*s["lengths"]):
        step = max(1, min(lq, (1 << 28) // lk))
        for head in range(h):
            keys = slice(kb, kb + lk)
            k, v = (s[x][keys, head // per].double() for x in "kv")
            for b in range(0, lq, step):
                rows = slice(qb + b, qb + min(lq, b + step))
                leaves = [x.contiguous().requires_grad_(grad) for x in (s["q"][rows, head].double(), k, v)]
                with torch.set_grad_enabled(grad):
                    z = leaves[0] @ leaves[1].t() / math.sqrt(d)
                    if case["causal"]:
                        seen = torch.ones(z.shape, device="cuda", dtype=torch.bool).tril(lk - lq + b)
                        z = z.where(seen, -math.inf)
                    o = torch.softmax(z, 1) @ leaves[2]
                out["out"][rows, head] = o.detach()
                out["lse"][rows, head] = torch.logsumexp(z.detach(), 1)
                if grad:
                    got = torch.autograd.grad(o, leaves, s["dout"][rows, head].double())
                    out["dq"][rows, head] = got[0]
                    out["dk"][keys, head // per] += got[1]
                    out["dv"][keys, head // per] += got[2]
        qb, kb = qb + lq, kb + lk
    return out


def exact(case, seed):
    return {"clip": _exact_clip, "qk": _exact_qk, "attention": _exact_attention}[case["op"]](prepare(case, seed))
