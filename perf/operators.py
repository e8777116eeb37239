"""The operators of the training path (attention with its backward pass, rotary positions with
several axes, norms fused with gate and residual, gradient norm and clipping) as cases that can
be timed and compared: `run` computes them in elementary torch operations in 32 bits, or, where
`own` is true, through the framework's entry points.

Sizes are those of the flow model (hidden 1024, 16 heads of 64, a 16 x 16 x 32 grid plus one
camera token = 8193 tokens, 1374 condition tokens, batch 2 for guidance) and of its small form
(hidden 128, 2 heads, 65 tokens, 17 condition tokens), and generic ones around them.
"""
import math
import os
import sys

import torch

own = False

F32 = torch.float32
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a training pass of the small model's cross-attention: launch latency
        {"name": "attn cross 65x17", "op": "attention", "b": 2, "h": 2, "lq": 65, "lk": 17, "bias": "none"},
        # latents against the padded condition tokens of two requests, one of them without any
        {"name": "attn cross 2049x1374 pad", "op": "attention", "b": 2, "h": 16, "lq": 2049, "lk": 1374,
         "bias": "empty"},
        # the flow model's self-attention at full size, batch 2
        {"name": "attn self 8193", "op": "attention", "b": 2, "h": 16, "lq": 8193, "lk": 8193, "bias": "none"},
        # one pooled query per request over the whole grid
        {"name": "attn one query 8193", "op": "attention", "b": 2, "h": 16, "lq": 1, "lk": 8193, "bias": "padding"},
        # rotation of a small prompt's queries and keys when serving: launch latency
        {"name": "rope 65 serve", "op": "rope", "b": 2, "l": 65, "h": 4, "d": 64, "pairs": "10,11,11",
         "grid": 32, "layout": "interleaved", "norm": True, "train": False, "dtype": "f32"},
        # queries and keys of the full grid, rotation and per-head norm, forward and backward
        {"name": "rope 8193 train", "op": "rope", "b": 2, "l": 8193, "h": 32, "d": 64, "pairs": "10,11,11",
         "grid": 32, "layout": "interleaved", "norm": True, "train": True, "dtype": "f32"},
        # video tokens (time, height, width) in 16 bits, wider heads, no norm
        {"name": "rope video bf16", "op": "rope", "b": 1, "l": 5985, "h": 24, "d": 128, "pairs": "16,24,24",
         "grid": 64, "layout": "halves", "norm": False, "train": True, "dtype": "bf16"},
        # the small model's block when serving
        {"name": "norm 65x128 serve", "op": "norm", "b": 2, "l": 65, "c": 128, "pre": "layer", "post": "none",
         "weights": False, "mod": True, "train": False, "dtype": "f32"},
        # the flow model's block at full size, forward and backward
        {"name": "norm 8193x1024 train", "op": "norm", "b": 2, "l": 8193, "c": 1024, "pre": "layer",
         "post": "rms", "weights": True, "mod": True, "train": True, "dtype": "f32"},
        # a ragged width in 16 bits
        {"name": "norm 2051x1111 bf16", "op": "norm", "b": 3, "l": 2051, "c": 1111, "pre": "rms", "post": "layer",
         "weights": True, "mod": True, "train": True, "dtype": "bf16"},
        # tables and gains of the small model
        {"name": "clip small", "op": "clip", "tensors": "small", "count": 10, "most": 768, "dtype": "f32"},
        # weights, biases, tables and gains of 28 blocks
        {"name": "clip 28 blocks", "op": "clip", "tensors": "model", "count": 476, "most": 0, "dtype": "f32"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "rope", "norm", "clip"])
    if op == "attention":
        return {"op": op, "b": rng.choice([1, 2]), "h": _log(rng, 2, 16), "lq": _log(rng, 1, 8193),
                "lk": _log(rng, 1, 8193), "bias": rng.choice(["none", "padding", "empty"])}
    if op == "rope":
        d = rng.choice([32, 64, 72, 96, 128])
        axes = rng.choice([1, 2, 3])
        pairs = [d // 2 // axes] * axes
        pairs[-1] += rng.choice([0, d // 2 - sum(pairs)])
        return {"op": op, "b": rng.choice([1, 2]), "l": _log(rng, 1, 8193), "h": _log(rng, 2, 32), "d": d,
                "pairs": ",".join(map(str, pairs)), "grid": rng.choice([16, 32, 64]),
                "layout": rng.choice(["interleaved", "halves"]), "norm": rng.random() < 0.5,
                "train": rng.random() < 0.7, "dtype": rng.choice(["f32", "bf16", "f16"])}
    if op == "norm":
        return {"op": op, "b": rng.choice([1, 2, 3]), "l": _log(rng, 1, 4097), "c": _log(rng, 64, 2048),
                "pre": rng.choice(["layer", "rms"]), "post": rng.choice(["none", "layer", "rms"]),
                "weights": rng.random() < 0.5, "mod": rng.random() < 0.7, "train": rng.random() < 0.7,
                "dtype": rng.choice(["f32", "bf16", "f16"])}
    return {"op": op, "tensors": "drawn", "count": _log(rng, 1, 400), "most": _log(rng, 16, 1 << 20),
            "dtype": rng.choice(["f32", "bf16"])}


# ----------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _prepare_attention(c, g):
    """Queries and keys as the per-head norm leaves them (unit elements), in the token-major layout
    of the projections; gradients at the scale of a mean loss."""
    b, h, lq, lk = c["b"], c["h"], c["lq"], c["lk"]
    q = _randn(g, b, lq, h, 64).transpose(1, 2)
    kv = _randn(g, b, lk, 2, h, 64)
    s = {"q": q, "k": kv[:, :, 0].transpose(1, 2), "v": (kv[:, :, 1] * 0.5).transpose(1, 2),
         "dout": _randn(g, b, lq, h, 64, scale=1e-3).transpose(1, 2), "bias": None}
    if c["bias"] != "none":  # each request's tokens end at its own length; a learned bias on the rest
        ends = torch.randint(max(1, lk // 2), lk + 1, (b, 1), generator=g, device="cuda")
        if c["bias"] == "empty":  # the last request has no key at all
            ends[-1] = 0
        j = torch.arange(lk, device="cuda")[None]
        s["bias"] = torch.where(j < ends, _randn(g, b, lk, scale=0.5), torch.full((), -math.inf, device="cuda"))
    return s


def _prepare_rope(c, g):
    """The query and key part of a packed projection, positions on a grid, frequencies of base 1e4."""
    dt = DTYPES[c["dtype"]]
    pairs = [int(p) for p in c["pairs"].split(",")]
    packed = _randn(g, c["b"], c["l"], c["h"] + c["h"] // 2, c["d"], dtype=dt)
    pos = torch.randint(0, c["grid"], (c["l"], len(pairs)), generator=g, device="cuda", dtype=torch.int32)
    inv = torch.cat([10000.0 ** (-torch.arange(p, dtype=torch.float64) / p) for p in pairs])
    s = {"x": packed[:, :, :c["h"]], "positions": pos, "inv_freq": inv.to(F32).cuda(), "pairs": pairs,
         "gamma": None, "dy": None}
    if c["norm"]:
        s["gamma"] = 1.0 + _randn(g, c["h"], c["d"], scale=0.02)
    if c["train"]:
        s["dy"] = _randn(g, c["b"], c["l"], c["h"], c["d"], scale=1e-3, dtype=dt)
    return s


def _prepare_norm(c, g):
    dt = DTYPES[c["dtype"]]
    b, l, w = c["b"], c["l"], c["c"]
    s = {"x": _randn(g, b, l, w, dtype=dt) + 0.25, "y": _randn(g, b, l, w, scale=0.5, dtype=dt)}
    for name in ("gate", "scale", "shift"):
        s[name] = _randn(g, b, w, scale=0.3) if c["mod"] else None
    for name, kind in (("pre_weight", c["pre"]), ("post_weight", c["post"])):
        s[name] = 1.0 + _randn(g, w, scale=0.1) if c["weights"] and kind != "none" else None
    if c["train"]:
        s["dz"], s["dh"] = (_randn(g, b, l, w, scale=1e-3, dtype=dt) for _ in range(2))
    return s


def _shapes(c):
    if c["tensors"] == "model":
        h = 1024
        block = [(h, h)] * 3 + [(2 * h, h), (4 * h, h), (h, 4 * h)] + [(h,)] * 4 + [(2 * h,), (4 * h,)]
        return (block + [(6, h)] + [(16, 64)] * 4) * 28
    if c["tensors"] == "small":
        return ([(6, 128)] + [(2, 64)] * 4) * 2
    # sizes between 1 and `most`, spread over their logarithm, by a rule of the index alone
    top = math.log(c["most"])
    return [(max(1, int(math.exp(top * ((i * 0.6180339887 + 0.37) % 1.0)))),) for i in range(c["count"])]


def _prepare_clip(c, g):
    """Gradients in tensors of their own; the clipped ones go side by side into one buffer, each on a
    256-byte boundary, so that they can be handed on whole."""
    dt = DTYPES[c["dtype"]]
    grads = [_randn(g, *shape, scale=1e-3, dtype=dt) for shape in _shapes(c)]
    ends, at = [], 0
    for t in grads:
        ends.append(at)
        at += (t.numel() + 127) // 128 * 128
    flat = torch.zeros(at, dtype=dt, device="cuda")
    return {"grads": grads, "flat": flat, "out": [flat[e:e + t.numel()].view(t.shape) for e, t in zip(ends, grads)],
            "max_norm": 0.05}


def prepare(case, seed):
    g = _gen(seed)
    make = {"attention": _prepare_attention, "rope": _prepare_rope, "norm": _prepare_norm, "clip": _prepare_clip}
    return {"case": case, **make[case["op"]](case, g)}


# ------------------------------------------------------------------------------ plain forms
def _plain_attention(s):
    q, k, v, do, bias = s["q"], s["k"], s["v"], s["dout"], s["bias"]
    sc = (q @ k.transpose(-1, -2)).mul_(0.125)
    if bias is not None:
        sc += bias[:, None, None, :]
    top = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, torch.ones_like(total), total)
    out = p @ v
    dv = p.transpose(-1, -2) @ do
    ds = (do @ v.transpose(-1, -2)).sub_((do * out).sum(-1, keepdim=True)).mul_(p)
    r = {"out": out, "dq": ds @ k * 0.125, "dk": ds.transpose(-1, -2) @ q * 0.125, "dv": dv}
    if bias is not None:
        r["dbias"] = ds.sum(2).sum(1)
    return r


def _turn(x, cos, sin, pairs, layout):
    """x [..., D] with its first 2 * pairs elements rotated pair by pair."""
    if layout == "interleaved":
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., 2 * pairs:]], -1)


def _plain_rope(s):
    c = s["case"]
    x, n, dt, d = s["x"].to(F32), sum(s["pairs"]), s["x"].dtype, c["d"]
    axis = torch.repeat_interleave(torch.arange(len(s["pairs"])), torch.tensor(s["pairs"])).cuda()
    angle = s["positions"].to(F32)[:, axis] * s["inv_freq"]
    cos, sin = angle.cos()[:, None, :], angle.sin()[:, None, :]
    r = _turn(x, cos, sin, n, c["layout"])
    gamma = s["gamma"]
    if gamma is not None:
        f = math.sqrt(d) / (r * r).sum(-1, keepdim=True).sqrt().clamp_min(1e-12)
    res = {"y": (r if gamma is None else r * f * gamma).to(dt)}
    if s["dy"] is not None:
        dr = dy = s["dy"].to(F32)
        if gamma is not None:
            res["dgamma"] = (dy * r * f).sum((0, 1))
            g = dy * gamma
            dr = f * (g - r * (r * g).sum(-1, keepdim=True) * (f * f / d))
        res["dx"] = _turn(dr, cos, -sin, n, c["layout"]).to(dt)
    return res


def _stats(v, kind):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = ((v * v).mean(-1, keepdim=True) + EPS).rsqrt()
    return v * r, r


def _unnorm(d, n, r, kind):
    """The gradient through n = norm(v), given the gradient d of n."""
    d = d - n * (d * n).mean(-1, keepdim=True)
    return r * (d - d.mean(-1, keepdim=True) if kind == "layer" else d)


def _one(t, like):
    return torch.ones((), device=like.device) if t is None else t


def _plain_norm(s):
    c = s["case"]
    x, y, dt = s["x"].to(F32), s["y"].to(F32), s["x"].dtype
    gate, scale, shift = (None if s[k] is None else s[k][:, None] for k in ("gate", "scale", "shift"))
    wq, wp = _one(s["post_weight"], x), _one(s["pre_weight"], x)
    m, rm = _stats(y, c["post"]) if c["post"] != "none" else (y, None)
    z = x + m * wq * _one(gate, x) * 0.5
    n, rn = _stats(z, c["pre"])
    u = n * wp
    h = u if scale is None else u * (1 + scale) + shift
    res = {"z": z.to(dt), "h": h.to(dt)}
    if c["train"]:
        dz, dh = s["dz"].to(F32), s["dh"].to(F32)
        du = dh if scale is None else dh * (1 + scale)
        dz = dz + _unnorm(du * wp, n, rn, c["pre"])
        dp = dz * _one(gate, x) * 0.5
        dm = dp * wq
        res["dx"] = dz.to(dt)
        res["dy"] = (dm if c["post"] == "none" else _unnorm(dm, m, rm, c["post"])).to(dt)
        if scale is not None:
            res["dscale"], res["dshift"], res["dgate"] = (dh * u).sum(1), dh.sum(1), (dz * m * wq).sum(1) * 0.5
        if s["pre_weight"] is not None:
            res["dpre_weight"] = (du * n).sum((0, 1))
        if s["post_weight"] is not None:
            res["dpost_weight"] = (dp * m).sum((0, 1))
    return res


def _plain_clip(s):
    norm = torch.stack([t.to(F32).square().sum() for t in s["grads"]]).sum().sqrt()
    c = (s["max_norm"] / (norm + 1e-6)).clamp_max(1.0)
    [o.copy_(t.to(F32) * c) for o, t in zip(s["out"], s["grads"])]
    return {"norm": norm, "grads": s["flat"]}


# ------------------------------------------------------------------- the framework's own calls
def _ops():
    path = os.path.join(os.getcwd(), "triposplat-cpu-avx512_b200")  # run from the repository's root
    if path not in sys.path:
        sys.path.insert(0, path)
    import train_ops

    return train_ops


def _own_attention(s):
    t = _ops()
    out, stats = t.attention_forward(s["q"], s["k"], s["v"], key_bias=s["bias"])
    dq, dk, dv, dbias = t.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, stats, key_bias=s["bias"])
    r = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if dbias is not None:
        r["dbias"] = dbias
    return r


def _own_rope(s):
    t = _ops()
    how = dict(axis_pairs=s["pairs"], gamma=s["gamma"], layout=s["case"]["layout"])
    r = {"y": t.axis_rope(s["x"], s["positions"], s["inv_freq"], **how)}
    if s["dy"] is not None:
        r["dx"], dgamma = t.axis_rope_backward(s["dy"], s["x"], s["positions"], s["inv_freq"], **how)
        if dgamma is not None:
            r["dgamma"] = dgamma
    return r


def _own_norm(s):
    t, c = _ops(), s["case"]
    how = dict(gate=s["gate"], scale=s["scale"], shift=s["shift"], pre=c["pre"], pre_weight=s["pre_weight"],
               post=None if c["post"] == "none" else c["post"], post_weight=s["post_weight"], residual_scale=0.5,
               eps=EPS)
    z, h, stats = t.norm_gate(s["x"], s["y"], **how)
    r = {"z": z, "h": h}
    if c["train"]:
        g = t.norm_gate_backward(s["dz"], s["dh"], s["x"], s["y"], stats, **how)
        r.update({"d" + k: v for k, v in g.items() if v is not None})
    return r


def _own_clip(s):
    return {"norm": _ops().clip_grad_norm(s["grads"], s["max_norm"], out=s["out"]), "grads": s["flat"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "rope": _own_rope, "norm": _own_norm, "clip": _own_clip}[op](state)
    return {"attention": _plain_attention, "rope": _plain_rope, "norm": _plain_norm, "clip": _plain_clip}[op](state)


# ------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "attention":
        # forward 2 and backward 5 products of lq x lk x 64 per head
        rows, keys = c["b"] * c["h"] * c["lq"], c["b"] * c["h"] * c["lk"]
        return {"bytes": 4 * 64 * (4 * rows + 4 * keys), "flops": 14.0 * 64 * rows * c["lk"]}
    if c["op"] == "rope":
        n = c["b"] * c["l"] * c["h"] * c["d"]
        each = (3 + (4 if c["norm"] else 0)) * (3 if c["train"] else 1)
        return {"bytes": SIZE[c["dtype"]] * n * (4 if c["train"] else 2), "flops": float(each * n)}
    if c["op"] == "norm":
        n = c["b"] * c["l"] * c["c"]
        return {"bytes": SIZE[c["dtype"]] * n * (8 if c["train"] else 4), "flops": (60.0 if c["train"] else 16.0) * n}
    n = sum(math.prod(s) for s in _shapes(c))
    return {"bytes": 2 * SIZE[c["dtype"]] * n, "flops": 3.0 * n}


# --------------------------------------------------------------- the definitions in 64 bits
def _exact_attention(s):
    """Head by head: softmax over the keys that exist, and the derivative of sum(out * dout) by the
    softmax's Jacobian."""
    b, h, lq, _ = s["q"].shape
    lk = s["k"].shape[2]
    r = {n: torch.zeros(b, h, l, 64, dtype=torch.float64, device="cuda")
         for n, l in (("out", lq), ("dq", lq), ("dk", lk), ("dv", lk))}
    if s["bias"] is not None:
        r["dbias"] = torch.zeros(b, lk, dtype=torch.float64, device="cuda")
    for i in range(b):
        keep = torch.arange(lk, device="cuda") if s["bias"] is None else (s["bias"][i] > -math.inf).nonzero()[:, 0]
        if not keep.numel():
            continue
        for j in range(h):
            q, do = s["q"][i, j].double(), s["dout"][i, j].double()
            k, v = s["k"][i, j][keep].double(), s["v"][i, j][keep].double()
            x = torch.einsum("id,jd->ij", q, k) / 8.0
            if s["bias"] is not None:
                x += s["bias"][i][keep].double()
            p = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
            dp = torch.einsum("id,jd->ij", do, v)
            ds = p * (dp - torch.einsum("ij,ij->i", p, dp)[:, None])
            r["out"][i, j] = torch.einsum("ij,jd->id", p, v)
            r["dv"][i, j, keep] = torch.einsum("ij,id->jd", p, do)
            r["dq"][i, j] = torch.einsum("ij,jd->id", ds, k) / 8.0
            r["dk"][i, j, keep] = torch.einsum("ij,id->jd", ds, q) / 8.0
            if s["bias"] is not None:
                r["dbias"][i, keep] += ds.sum(0)
    return r


def _exact_rope(s):
    """Pairs as complex numbers; the derivative by the product rule on x / |x|."""
    c = s["case"]
    n, d, b, l, h = sum(s["pairs"]), c["d"], c["b"], c["l"], c["h"]
    angle, at = [], 0
    for a, p in enumerate(s["pairs"]):
        angle.append(s["positions"][:, a].double()[:, None] * s["inv_freq"][at:at + p].double()[None])
        at += p
    turn = torch.polar(torch.ones(l, n, dtype=torch.float64, device="cuda"), torch.cat(angle, 1))[:, None]
    first = torch.arange(0, 2 * n, 2, device="cuda") if c["layout"] == "interleaved" else torch.arange(n, device="cuda")
    second = first + (1 if c["layout"] == "interleaved" else n)

    def rotate(x, by):
        w, out = torch.complex(x[..., first], x[..., second]) * by, x.clone()
        out[..., first], out[..., second] = w.real, w.imag
        return out

    r = rotate(s["x"].double(), turn)
    gamma = None if s["gamma"] is None else s["gamma"].double()
    length = torch.linalg.vector_norm(r, dim=-1, keepdim=True).clamp_min(1e-12)
    unit = r / length * math.sqrt(d)
    res = {"y": r if gamma is None else unit * gamma}
    if s["dy"] is not None:
        g = s["dy"].double()
        if gamma is not None:
            res["dgamma"] = torch.einsum("blhd,blhd->hd", g, unit)
            g = g * gamma * (math.sqrt(d) / length)
            g = g - (r / length) * torch.einsum("blhd,blhd->blh", g, r / length)[..., None]
        res["dx"] = rotate(g, turn.conj())
    return res


def _exact_norm(s):
    """The formulas in 64 bits, differentiated by autograd."""
    c = s["case"]
    leaf = {k: s[k].double().requires_grad_(c["train"])
            for k in ("x", "y", "gate", "scale", "shift", "pre_weight", "post_weight") if s[k] is not None}

    def norm(v, kind):
        if kind == "none":
            return v
        mean = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
        return (v - mean) / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + EPS)

    p = norm(leaf["y"], c["post"]) * leaf.get("post_weight", 1.0)
    z = leaf["x"] + 0.5 * p * (leaf["gate"][:, None] if "gate" in leaf else 1.0)
    h = norm(z, c["pre"]) * leaf.get("pre_weight", 1.0)
    if "scale" in leaf:
        h = h * (1.0 + leaf["scale"][:, None]) + leaf["shift"][:, None]
    res = {"z": z.detach(), "h": h.detach()}
    if c["train"]:
        got = torch.autograd.grad([z, h], list(leaf.values()), [s["dz"].double(), s["dh"].double()])
        res.update({"d" + k: t for k, t in zip(leaf, got)})
    return res


def _exact_clip(s):
    total = math.sqrt(math.fsum(float(torch.linalg.vector_norm(t.double())) ** 2 for t in s["grads"]))
    flat = torch.zeros(s["flat"].numel(), dtype=torch.float64, device="cuda")
    at = 0
    for t in s["grads"]:
        flat[at:at + t.numel()] = t.double().reshape(-1) * min(1.0, s["max_norm"] / (total + 1e-6))
        at += (t.numel() + 127) // 128 * 128
    return {"norm": torch.tensor(total, dtype=torch.float64), "grads": flat}


def exact(case, seed):
    s = prepare(case, seed)
    make = {"attention": _exact_attention, "rope": _exact_rope, "norm": _exact_norm, "clip": _exact_clip}
    with torch.enable_grad():
        return make[case["op"]](s)
