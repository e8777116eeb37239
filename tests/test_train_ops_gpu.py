"""Training operators (rotary positions, norm with gate, gradient clipping) against their
definitions in 64 bits, and gradients against central differences.

Tolerances.  u = 2^-24 is the rounding of fp32, U the rounding of the output's type (2^-24,
2^-8 for bf16, 2^-11 for fp16, each half the type's epsilon).  An output is at most a few
dozen fp32 roundings away from its definition, each relative to an intermediate no larger than
the row's scale: |err| <= U |ref| (1 + 2^-6) + 64 u S, with S that scale.  A column sum of n terms
t adds errors of single terms (up to 64 u |t|) and of at most n sequential additions (u times a partial
sum): |err| <= (64 + n) u sum|t|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = {t: torch.finfo(t).eps / 2 for t in TYPES}


def randn(seed, *shape, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float64) * scale).to(dtype)


def near(got, ref, scale, dtype=torch.float32):
    """|got - ref| within U |ref| and 64 u of `scale` (and the type's smallest step)."""
    got, bound = got.double(), UNIT[dtype] * ref.abs() * (1 + 2.0 ** -6) + 64 * U32 * scale
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25
    assert torch.isfinite(got).all()
    worst = ((got - ref).abs() - bound).max().item()
    assert worst <= 0, f"beyond its bound by {worst:.3e} (bound up to {bound.max().item():.3e})"


def near_sum(got, terms, dims):
    """A column sum against the 64-bit sum of `terms` over `dims`."""
    n = math.prod(terms.shape[d] for d in dims)
    ref, mass = terms.sum(dims), terms.abs().sum(dims)
    assert ((got.double() - ref).abs() <= (64 + n) * U32 * mass + 1e-300).all()


# ---------------------------------------------------------------------------- rotary positions
def rope_ref(x, pos, inv, pairs, layout, gamma):
    """(r, n, y): rotated vector, its length, the output, in 64 bits; pos [B, L, axes]."""
    axis = [a for a, p in enumerate(pairs) for _ in range(p)]
    n = len(axis)
    ang = pos[..., axis].double() * inv.double()
    c, s = ang.cos()[:, :, None], ang.sin()[:, :, None]
    i = torch.arange(n, device=x.device)
    i, j = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, n + i)
    r = x.double().clone()
    a, b = x.double()[..., i], x.double()[..., j]
    r[..., i], r[..., j] = a * c - b * s, a * s + b * c
    length = r.norm(dim=-1, keepdim=True)
    y = r if gamma is None else r * math.sqrt(x.shape[-1]) / length.clamp_min(1e-12) * gamma.double()
    return r, length, y, (lambda v: unturn(v, c, s, i, j))


def unturn(v, c, s, i, j):
    o = v.clone()
    o[..., i], o[..., j] = v[..., i] * c + v[..., j] * s, v[..., j] * c - v[..., i] * s
    return o


ROPE = [(1, 1, 1, 2, [1], "interleaved"), (2, 65, 4, 64, [10, 11, 11], "interleaved"), (1, 33, 3, 64, [5, 0, 9], "halves"),
        (2, 31, 5, 72, [12, 12, 12], "halves"), (1, 97, 2, 256, [128], "interleaved"), (1, 40, 9, 128, [16, 24, 24], "halves"),
        (3, 5, 1, 6, [1, 1], "interleaved"), (1, 1025, 2, 64, [8, 8, 8, 8], "interleaved")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("case", ROPE, ids=str)
def test_rope(case, norm, dtype):
    import train_ops

    B, L, H, D, pairs, layout = case
    packed = randn(1, B, L, H + 2, D, dtype=dtype)
    x = packed[:, :, 1:H + 1]  # strided: heads of a wider projection
    dy = randn(2, B, H, L, D, dtype=dtype).transpose(1, 2)
    gamma = 1 + randn(3, H, D, scale=0.1) if norm else None
    inv = torch.cat([10000.0 ** (-torch.arange(p) / max(p, 1)) for p in pairs]).float().cuda()
    pos = torch.randint(0, 2000, (B, L, len(pairs)), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    how = dict(axis_pairs=pairs, gamma=gamma, layout=layout)
    y = train_ops.axis_rope(x, pos, inv, **how)
    dx, dgamma = train_ops.axis_rope_backward(dy, x, pos, inv, **how)
    r, n, ref, back = rope_ref(x, pos, inv, pairs, layout, gamma)
    f = math.sqrt(D) / n.clamp_min(1e-12)
    near(y, ref, (f * n * gamma.double().abs().amax(-1, keepdim=True)) if norm else n, dtype)
    g = dy.double()
    if norm:
        near_sum(dgamma, g * r * f, (0, 1))
        g = g * gamma.double()
        near(dx, back(f * (g - r * (r * g).sum(-1, keepdim=True) / n ** 2)), f * g.norm(dim=-1, keepdim=True), dtype)
    else:
        assert dgamma is None
        near(dx, back(g), g.norm(dim=-1, keepdim=True), dtype)


def test_rope_positions():
    """Shared and per-entry positions in all three types, far from zero, and in place."""
    import train_ops

    x, inv = randn(1, 2, 9, 2, 64), (10000.0 ** (-torch.arange(32) / 32)).float().cuda()
    for pos in (torch.arange(9, device="cuda")[:, None] * 12345 + 10 ** 6, torch.full((9, 1), -2 ** 40 + 7, device="cuda")):
        _, n, ref, _ = rope_ref(x, pos.expand(2, 9, 1), inv, [32], "interleaved", None)
        # cosine of an angle formed in 64 bits: its own rounding is 2^-53 of the angle
        slack = n * pos.abs().max().item() * 2.0 ** -52
        kinds = [torch.int64] + ([torch.int32, torch.float32] if pos.abs().max() < 2 ** 24 else [])
        for kind in kinds:
            y = train_ops.axis_rope(x, pos.to(kind), inv, axis_pairs=[32])
            assert ((y.double() - ref).abs() <= 64 * U32 * n + slack).all()
            assert torch.equal(y, train_ops.axis_rope(x, pos.to(kind).expand(2, 9, 1), inv, axis_pairs=[32]))
    z = x.clone()
    assert train_ops.axis_rope(z, pos, inv, axis_pairs=[32], out=z) is z and torch.equal(z, y)


def test_rope_matches_the_table_form():
    """The flow model's table of cosines and its rope + norm kernels, on its own grid."""
    import native_ops
    import train_ops
    from flow_model import FlowSpec, rope_freqs

    s = FlowSpec.small()
    x = randn(5, 1, s.seq, s.heads, 64)
    gamma = 1 + randn(6, s.heads, 64, scale=0.02)
    gx, gy, gz = s.grid
    n = torch.arange(s.latent_tokens)
    pos = torch.stack([n // (gy * gz), (n // gz) % gy, n % gz], 1)
    pos = torch.cat([pos, torch.zeros(1, 3, dtype=pos.dtype)]).int().cuda()  # the camera token is unrotated
    inv = torch.cat([1.0 / s.theta ** (torch.arange(p, dtype=torch.float64) / p) for p in s.rope_pairs]).float().cuda()
    y = train_ops.axis_rope(x, pos, inv, axis_pairs=s.rope_pairs, gamma=gamma)
    table = torch.from_numpy(rope_freqs(s)).cuda()
    ref = native_ops.multihead_rmsnorm(native_ops.rope_complex(x, table), gamma)
    # inv_freq in fp32: an angle of up to 4 rad is off by 4 * 2^-24; outputs are up to 8 |gamma|
    assert (y - ref).abs().max().item() <= 16 * 64 * U32


def test_rope_vanishing_vectors():
    """A zero vector stays zero, forward and backward finite; below the norm's floor the output is linear."""
    import train_ops

    x = torch.zeros(1, 2, 1, 64, device="cuda")
    x[0, 1] = 1e-14
    inv, pos = torch.ones(32, device="cuda"), torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    gamma, dy = torch.ones(1, 64, device="cuda"), randn(1, 1, 2, 1, 64)
    y = train_ops.axis_rope(x, pos, inv, axis_pairs=[32], gamma=gamma)
    assert torch.equal(y[0, 0], torch.zeros_like(y[0, 0]))
    near(y[0, 1], x[0, 1].double() * 8e12, 1.0)
    dx, _ = train_ops.axis_rope_backward(dy, x, pos, inv, axis_pairs=[32], gamma=gamma)
    near(dx, dy.double() * 8e12, 8e12)


# -------------------------------------------------------------------------- norms with gate
def norm_ref(x, y, p, pre, post, rho, eps):
    """z, h in 64 bits (autograd leaves allowed)."""
    def norm(v, kind):
        if kind is None:
            return v
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        return v / (v.square().mean(-1, keepdim=True) + eps).sqrt()

    one = torch.ones((), dtype=torch.float64, device=x.device)
    row = {k: one if p.get(k) is None else p[k][:, None] if p[k].dim() == 2 else p[k]
           for k in ("gate", "scale", "shift", "pre_weight", "post_weight")}
    z = x + rho * row["gate"] * row["post_weight"] * norm(y, post)
    if pre is None:
        return z, None
    h = norm(z, pre) * row["pre_weight"]
    return z, h if p.get("scale") is None else h * (1 + row["scale"]) + row["shift"]


NORM = [(1, 1, 1), (2, 65, 128), (3, 7, 1111), (2, 130, 1024), (1, 3, 8192), (1, 2, 4100), (5, 33, 96), (1, 700, 40)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kinds", [("layer", None), ("layer", "rms"), ("rms", "layer"), (None, "rms")], ids=str)
@pytest.mark.parametrize("case", NORM, ids=str)
def test_norm_gate(case, kinds, dtype):
    import train_ops

    B, L, C = case
    pre, post = kinds
    full = (B + L + C) % 2 == 0  # every parameter, or none
    x = (randn(1, B, L + 1, C, dtype=dtype) + 0.5)[:, 1:]
    y = randn(2, L, B, C, dtype=dtype).transpose(0, 1)
    p = dict(gate=randn(3, B, C), scale=randn(4, B, C, scale=0.3) if pre else None, shift=randn(5, B, C) if pre else None,
             pre_weight=1 + randn(6, C, scale=0.1) if pre else None,
             post_weight=1 + randn(7, C, scale=0.1) if post else None) if full else {}
    how = dict(p, pre=pre, post=post, residual_scale=0.7, eps=1e-5)
    z, h, stats = train_ops.norm_gate(x, y, **how)
    dz, dh = randn(8, B, L, C, dtype=dtype), randn(9, B, L, C, dtype=dtype) if pre else None
    got = train_ops.norm_gate_backward(dz, dh, x, y, stats, **how)
    leaf = {k: v.double().requires_grad_() for k, v in dict(p, x=x, y=y).items() if v is not None}
    rz, rh = norm_ref(leaf["x"], leaf["y"], leaf, pre, post, 0.7, 1e-5)
    # scales: |z| up to |x| and the gated norm; h carries the error of z through 1 / std
    top = lambda v: v.detach().abs().amax(-1, keepdim=True)  # noqa: E731
    big = lambda k: p[k].abs().max().double() if p.get(k) is not None else 1.0  # noqa: E731
    m = norm_ref(x.double() * 0, y.double(), {}, None, post, 1.0, 1e-5)[0]
    zs = top(x.double()) + 0.7 * big("gate") * big("post_weight") * (top(m) + (1 if post else 0))
    near(z, rz.detach(), zs, dtype)
    if pre:
        v = rz.detach()
        v = v - v.mean(-1, keepdim=True) if pre == "layer" else v
        r = 1 / (v.square().mean(-1, keepdim=True) + 1e-5).sqrt()
        hs = (r * zs + top(v) * r) * big("pre_weight") * (1 + big("scale")) * (1 + r * zs / math.sqrt(C)) + big("shift")
        near(h, rh.detach(), hs, dtype)
    else:
        assert h is None
    loss = (rz * dz.double()).sum() + ((rh * dh.double()).sum() if pre else 0)
    ref = dict(zip(leaf, torch.autograd.grad(loss, list(leaf.values()))))
    # gradients of x: the row's largest dh through r (its norm's derivative has norm <= 1, the
    # error of n is that of h), and dz
    gs = top(dz.double())
    if pre:
        gs = gs + r * hs / (1 + big("shift")) * top(dh.double()) * big("pre_weight") * (1 + big("scale")) * (1 + hs)
    near(got["x"], ref["x"], gs, dtype)
    ry = 1.0
    if post:
        v = y.double()
        v = v - v.mean(-1, keepdim=True) if post == "layer" else v
        ry = 1 / (v.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    near(got["y"], ref["y"], gs * 0.7 * big("gate") * big("post_weight") * ry * (1 + top(m)) ** 2 * (1 + ry * top(y.double())), dtype)
    n = L * (1 if full else 0)
    for k in ("gate", "scale", "shift", "pre_weight", "post_weight"):
        if p.get(k) is None:
            assert got[k] is None
            continue
        # every term of the sum is at most (row scale of its factors); n of them, in order
        rows = (gs * (1 + top(m)) * big("gate") * big("post_weight") if k in ("gate", "post_weight")
                else top(dh.double()) * (1 + hs) * (1 + big("scale")) * big("pre_weight"))
        mass = rows.sum(1)[:, 0] if ref[k].dim() == 2 else rows.sum()
        mass = mass[:, None] if ref[k].dim() == 2 else mass
        assert ((got[k].double() - ref[k]).abs() <= (64 + n) * U32 * mass).all(), k


def test_norm_gate_half_of_the_gradients():
    """Either incoming gradient alone; they add up to both (fp32, linear in dz and dh)."""
    import train_ops

    x, y, dz, dh = (randn(s, 2, 50, 96) for s in range(4))
    how = dict(gate=randn(5, 2, 96), pre="layer", post="rms")
    _, _, stats = train_ops.norm_gate(x, y, **how)
    both, a, b = (train_ops.norm_gate_backward(u, v, x, y, stats, **how) for u, v in ((dz, dh), (dz, None), (None, dh)))
    for k in ("x", "y", "gate"):
        assert (a[k] + b[k] - both[k]).abs().max().item() <= 256 * U32 * both[k].abs().max().item()


def test_norm_gate_differences():
    """<gradient, direction> against central differences of the kernel's own forward pass.  A step
    of 2^-6 leaves an error of its square times a third derivative of order one, and fp32 rounding of
    the outputs over the step: 2e-3 of the derivative's scale covers both."""
    import train_ops

    B, L, C = 2, 17, 72
    t = {k: randn(i, B, L, C) for i, k in enumerate(("x", "y", "dz", "dh"))}
    p = dict(gate=randn(5, B, C), scale=randn(6, B, C, scale=0.3), shift=randn(7, B, C),
             pre_weight=1 + randn(8, C, scale=0.1), post_weight=1 + randn(9, C, scale=0.1))
    kw = dict(pre="layer", post="rms", residual_scale=0.6)

    def value(x, y, q):
        z, h, _ = train_ops.norm_gate(x, y, **q, **kw)
        return ((z.double() * t["dz"].double()).sum() + (h.double() * t["dh"].double()).sum()).item()

    _, _, stats = train_ops.norm_gate(t["x"], t["y"], **p, **kw)
    g = train_ops.norm_gate_backward(t["dz"], t["dh"], t["x"], t["y"], stats, **p, **kw)
    for i, k in enumerate(("x", "y", *p)):
        base = dict(p, x=t["x"], y=t["y"])
        d = randn(20 + i, *base[k].shape)
        step = 2.0 ** -6
        side = []
        for sign in (1, -1):
            q = dict(base, **{k: base[k] + sign * step * d})
            side.append(value(q.pop("x"), q.pop("y"), q))
        told = (g[k].double() * d.double()).sum().item()
        scale = g[k].double().norm().item() * d.double().norm().item()
        assert abs((side[0] - side[1]) / (2 * step) - told) <= 2e-3 * scale, k


def test_rope_differences():
    """As above for the rotation with its norm."""
    import train_ops

    x, dy, gamma = randn(1, 2, 9, 3, 64), randn(2, 2, 9, 3, 64), 1 + randn(3, 3, 64, scale=0.1)
    inv, pos = torch.rand(30, device="cuda"), torch.randint(0, 50, (9, 2), device="cuda")
    how = dict(axis_pairs=[10, 20], layout="halves")
    dx, dgamma = train_ops.axis_rope_backward(dy, x, pos, inv, gamma=gamma, **how)

    def value(x, gamma):
        return (train_ops.axis_rope(x, pos, inv, gamma=gamma, **how).double() * dy.double()).sum().item()

    step = 2.0 ** -6
    for g, d, at in ((dx, randn(4, 2, 9, 3, 64), lambda s: (x + s * step * d, gamma)),
                     (dgamma, randn(5, 3, 64), lambda s: (x, gamma + s * step * d))):
        told = (g.double() * d.double()).sum().item()
        scale = g.double().norm().item() * d.double().norm().item()
        assert abs((value(*at(1)) - value(*at(-1))) / (2 * step) - told) <= 2e-3 * scale


# ------------------------------------------------------------------------------- clipping
@pytest.mark.parametrize("sizes", [[1], [0, 3], [5, 8192, 8193, 20000], [7] * 900, [100003, 1, 64] * 30], ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("dtypes", [TYPES[:1], TYPES], ids=["f32", "mixed"])
def test_clip(sizes, dtypes):
    """Norm to half a unit of fp32 and the roundings of the square root; every element to the scale's
    few fp32 roundings and its own type's.  In place and into outputs, clipped and not."""
    import train_ops

    buf = [randn(i, n + 1, dtype=dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]
    grads = [b[i % 2:i % 2 + n] for i, (b, n) in enumerate(zip(buf, sizes))]  # every other one misaligned
    total = math.sqrt(sum(g.double().square().sum().item() for g in grads))
    for max_norm in (total * 0.1, total * 10, 0.0):
        outs = [torch.empty_like(g) for g in grads]
        norm = train_ops.clip_grad_norm(grads, max_norm, out=outs)
        assert norm.dtype == torch.float32 and abs(norm.item() - total) <= 4 * U32 * total
        c = min(1.0, max_norm / (total + 1e-6))
        for g, o in zip(grads, outs):
            if g.numel():
                near(o, g.double() * c, (g.double() * c).abs(), g.dtype)
            if c == 1.0:
                assert torch.equal(g, o)
        here = [b.clone() for b in buf]
        view = [h[i % 2:i % 2 + n] for i, (h, n) in enumerate(zip(here, sizes))]
        assert torch.equal(train_ops.clip_grad_norm(view, max_norm), norm)
        assert all(torch.equal(a, b) for a, b in zip(view, outs))
        for i, (h, b, n) in enumerate(zip(here, buf, sizes)):  # nothing beside the views is written
            assert torch.equal(h[:i % 2], b[:i % 2]) and torch.equal(h[i % 2 + n:], b[i % 2 + n:])


def test_clip_extremes():
    """Squares beyond fp32's range, and norms that are not finite."""
    import train_ops

    big = torch.full((1000,), 1e30, device="cuda")
    norm = train_ops.clip_grad_norm([big], 1.0)
    assert abs(norm.item() / (math.sqrt(1000) * 1e30) - 1) < 4 * U32 and abs(big[0].item() * math.sqrt(1000) - 1) < 8 * U32
    small = torch.full((1000,), 1e-30, device="cuda")
    assert abs(train_ops.clip_grad_norm([small], 1.0).item() / (math.sqrt(1000) * 1e-30) - 1) < 4 * U32
    for bad in (math.inf, math.nan):
        g = torch.ones(70, device="cuda")
        g[3] = bad
        ref = g * (1.0 / (torch.tensor(bad) + 1e-6)).item() if bad != bad else g * 0.0
        norm = train_ops.clip_grad_norm([g], 1.0)
        assert torch.equal(norm.isnan().cpu(), torch.tensor(bad != bad)) and torch.equal(g.isnan(), ref.isnan())


# --------------------------------------------------------------- streams, order, refusals
def test_repeatable_on_a_side_stream():
    """The same bits on another stream as on the default one, and on every run."""
    import train_ops

    x, y, dz = (randn(s, 2, 300, 256) for s in range(3))
    gate = randn(4, 2, 256)
    heads, gamma = randn(5, 2, 300, 4, 64), randn(6, 4, 64)
    pos, inv = torch.arange(300, device="cuda")[:, None], torch.rand(32, device="cuda")

    def all_of():
        z, h, st = train_ops.norm_gate(x, y, gate=gate, post="rms")
        g = train_ops.norm_gate_backward(dz, dz, x, y, st, gate=gate, post="rms")
        r = train_ops.axis_rope_backward(heads, heads, pos, inv, axis_pairs=[32], gamma=gamma)
        outs = [torch.empty_like(dz)]
        return [z, h, g["x"], g["y"], g["gate"], *r, train_ops.clip_grad_norm([dz], 0.1, out=outs), *outs]

    first = all_of()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = all_of()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_refusals():
    import train_ops

    x, inv = randn(1, 1, 4, 2, 64), torch.ones(32, device="cuda")
    pos, r = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), train_ops.axis_rope
    for call in (lambda: r(x[0], pos, inv, axis_pairs=[32]), lambda: r(x.double(), pos, inv, axis_pairs=[32]),
                 lambda: r(x[..., :63], pos, inv, axis_pairs=[31]), lambda: r(x, pos, inv, axis_pairs=[33]),
                 lambda: r(x, pos, inv[:31], axis_pairs=[32]), lambda: r(x, pos[:3], inv, axis_pairs=[32]),
                 lambda: r(x, pos.half(), inv, axis_pairs=[32]), lambda: r(x, pos.cpu(), inv, axis_pairs=[32]),
                 lambda: r(x, pos, inv, axis_pairs=[32], layout="pairs"), lambda: r(x, pos, inv, axis_pairs=[]),
                 lambda: r(x, pos, inv, axis_pairs=[32], gamma=torch.ones(2, 63, device="cuda")),
                 lambda: r(x, pos, inv, axis_pairs=[32], out=x.half()), lambda: r(x.cpu(), pos.cpu(), inv.cpu(), axis_pairs=[32]),
                 lambda: r(x, pos, inv, axis_pairs=[32], out=x[:, :1].expand(1, 4, 2, 64))):
        with pytest.raises(ValueError):
            call()
    t, n = randn(2, 2, 3, 8), train_ops.norm_gate
    w = torch.ones(8, device="cuda")
    for call in (lambda: n(t, t[:1]), lambda: n(t, t.half()), lambda: n(t[0], t[0]), lambda: n(t, t, pre="batch"),
                 lambda: n(t, t, scale=t[:, 0]), lambda: n(t, t, pre=None, pre_weight=w), lambda: n(t, t, post_weight=w),
                 lambda: n(t, t, gate=w), lambda: n(t, t, gate=t[:, 0].half()), lambda: n(randn(1, 1, 1, 8193), randn(1, 1, 1, 8193)),
                 lambda: n(t[:, :0], t[:, :0]),
                 lambda: train_ops.norm_gate_backward(None, None, t, t, torch.zeros(2, 3, 4, device="cuda")),
                 lambda: train_ops.norm_gate_backward(t, t, t, t, torch.zeros(2, 3, 4, device="cuda"), pre=None)):
        with pytest.raises(ValueError):
            call()
    c = train_ops.clip_grad_norm
    for call in (lambda: c([], 1.0), lambda: c([t], -1.0), lambda: c([t], math.nan), lambda: c([t.double()], 1.0),
                 lambda: c([t[..., ::2]], 1.0), lambda: c([t], 1.0, out=[]), lambda: c([t], 1.0, out=[t.half()]),
                 lambda: c([t, t.cpu()], 1.0)):
        with pytest.raises(ValueError):
            call()
