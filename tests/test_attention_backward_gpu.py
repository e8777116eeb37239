"""Attention for training (forward with statistics, backward) against its definition in 64 bits.

Tolerances.  Every product is formed from fp16 pairs of 22 bits with the lowest partial product
left out, so a score is off by at most 3 * 2^-22 sum|q k| / 8 and a probability by that, relative.
The tests' scores have sum|q k| / 8 of about 64 * 0.64 / 8 = 5 (unit normal q, k), worst rows three
times that: 15 * 3 * 2^-22 = 1.1e-5 at the very worst, some 1e-6 root mean square, and gradients
are sums of products of probabilities with factors of the same accuracy.  Bounds: 2-norm of the error
within 2e-6 of the result's, largest error within 4e-5 of its root mean square or of the value.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

REL, TOP = 2e-6, 4e-5


def randn(seed, *shape, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda") * scale


def near(got, ref, name="", floor=0.0):
    """`floor`: a level below which a result is rounding (sums that cancel)."""
    got, err = got.double(), (got.double() - ref).abs()
    assert torch.isfinite(got).all(), name
    rms = max(ref.square().mean().sqrt().item(), floor)
    if rms == 0.0:
        assert err.max().item() == 0.0, name
        return
    assert err.square().mean().sqrt().item() <= REL * rms, f"{name}: rel {err.square().mean().sqrt().item() / rms:.2e}"
    worst = (err / ref.abs().clamp_min(rms)).max().item()
    assert worst <= TOP, f"{name}: max {worst:.2e}"


def reference(q, k, v, do, bias=None, scores=True):
    """out, dq, dk, dv, ds in 64 bits; bias [B, H, Lk], keys at -inf left out (their rows zeroed)."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    b = torch.zeros((*k.shape[:3],), dtype=torch.float64, device=k.device) if bias is None else bias.double()
    gone = b == -math.inf
    k, v = k.masked_fill(gone[..., None], 0), v.masked_fill(gone[..., None], 0)
    top = b.amax(-1, keepdim=True)
    x = (q @ k.mT / 8 if scores else 0 * (q @ k.mT)) + (b - torch.where(top == -math.inf, 0.0, top))[:, :, None]
    m = x.amax(-1, keepdim=True)
    e = (x - torch.where(m == -math.inf, 0.0, m)).exp()
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    out = p @ v
    ds = p * (do @ v.mT - (do * out).sum(-1, keepdim=True))
    return out, ds @ k / 8, ds.mT @ q / 8, p.mT @ do, ds


def both(q, k, v, do, key_bias=None, **how):
    import train_ops

    out, stats = train_ops.attention_forward(q, k, v, key_bias=key_bias)
    return out, *train_ops.attention_backward(do, q, k, v, out, stats, key_bias=key_bias, **how)


SIZES = [(1, 1, 1, 1), (1, 2, 1, 700), (2, 1, 700, 1), (1, 3, 63, 65), (2, 2, 64, 64), (1, 2, 65, 17), (1, 2, 127, 129),
         (1, 1, 128, 128), (2, 3, 129, 191), (1, 2, 193, 1030), (1, 5, 1025, 257), (3, 60, 130, 140)]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size):
    B, H, Lq, Lk = size
    qkv = randn(1, B, Lk, 3, H, 64)  # token-major, sliced from one projection
    q, k, v = randn(2, B, Lq, H, 64).transpose(1, 2), qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
    do = randn(3, B, H, Lq, 64, scale=1e-3)
    out, dq, dk, dv, db = both(q, k, v, do)
    ref = reference(q, k, v, do)
    assert db is None
    # with one key ds cancels to rounding: measured against the terms it cancels from, Lq of them in dk
    floor = (do.double().norm(dim=-1).mean() * v.double().norm(dim=-1).mean() / 64).item() if Lk == 1 else 0.0
    floors = {"dq": floor, "dk": floor * math.sqrt(Lq)}
    for name, a, b in zip(("out", "dq", "dk", "dv"), (out, dq, dk, dv), ref):
        near(a, b, name, floors.get(name, 0.0))


@pytest.mark.parametrize("shape", ["keys", "batch", "head"])
def test_bias_and_its_gradient(shape):
    """A bias with missing keys, in its three shapes; what the missing keys hold is not read."""
    B, H, Lq, Lk = 2, 3, 150, 333
    q, do = randn(1, B, H, Lq, 64), randn(2, B, H, Lq, 64, scale=1e-3)
    k, v = randn(3, B, H, Lk, 64), randn(4, B, H, Lk, 64)
    full = {"keys": (Lk,), "batch": (B, Lk), "head": (B, H, Lk)}[shape]
    bias = randn(5, *full)
    gone = torch.rand(full, device="cuda", generator=torch.Generator("cuda").manual_seed(6)) < 0.4
    bias[gone] = -math.inf
    wide = {"keys": bias[None, None], "batch": bias[:, None], "head": bias}[shape].expand(B, H, Lk)
    ref = reference(q, k, v, do, wide)
    hole = wide == -math.inf
    for fill in (math.nan, math.inf, 0.0):
        kk, vv = k.masked_fill(hole[..., None], fill), v.masked_fill(hole[..., None], fill)
        out, dq, dk, dv, db = both(q, kk, vv, do, bias)
        for name, a, b in zip(("out", "dq", "dk", "dv"), (out, dq, dk, dv), ref):
            near(a, b, name)
        assert not dk[hole].any() and not dv[hole].any()
        ds = ref[4].sum(2)
        near(db, {"keys": ds.sum((0, 1)), "batch": ds.sum(1), "head": ds}[shape], "dbias")
        assert db.shape == bias.shape and not db[gone].any()
    assert both(q, k, v, do, bias, bias_grad=False)[4] is None


def test_rows_without_keys():
    """One batch entry with no key at all: zeros, forward and backward; the other as without it."""
    B, H, Lq, Lk = 2, 2, 70, 200
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    bias = torch.zeros(B, Lk, device="cuda")
    bias[1] = -math.inf
    got = both(q, k, v, do, bias)
    for t in got:
        assert not t[1].any() and torch.isfinite(t).all()
    alone = both(q[:1], k[:1], v[:1], do[:1])
    for a, b in zip(got[:4], alone[:4]):
        assert torch.equal(a[:1], b)


def test_lowest_values():
    """A mask of the type's lowest value: no weight beside other keys, the bias alone where every key has
    it (scores vanish beside it), and large common values cancel."""
    B, H, Lq, Lk = 1, 2, 40, 150
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    low = torch.finfo(torch.float32).min
    bias = torch.zeros(Lk, device="cuda")
    bias[50:] = low
    hidden = bias.masked_fill(bias == low, -math.inf)
    for a, b in zip(both(q, k, v, do, bias), both(q, k, v, do, hidden)):
        near(a, b.double(), floor=1e-30)
    bias[:] = low
    ref = reference(q, k, v, do, torch.zeros(B, H, Lk, device="cuda"), scores=False)
    got = both(q, k, v, do, bias)
    for a, b in zip(got[:4], ref):
        near(a, b)
    assert torch.equal(got[0], both(q, k, v, do, torch.full((Lk,), 2.0 ** 100, device="cuda"))[0])
    # up to what fp32 keeps of the scores beside it, a common value changes nothing
    near(both(q, k, v, do, torch.full((Lk,), -3.0e4, device="cuda"))[0], both(q, k, v, do)[0].double())


@pytest.mark.parametrize("what", ["peaked", "scaled", "uneven"])
def test_ranges(what):
    """Near one-hot rows, gradients and values far from one, rows of very different size."""
    B, H, Lq, Lk = 1, 2, 300, 520
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    bias = None
    if what == "peaked":
        # a dominant key per row through the bias (scores stay of unit size, as the tolerance assumes)
        bias = torch.zeros(Lk, device="cuda")
        bias[::97] = 12.0
    elif what == "scaled":
        do, v = do * 1e-12, v * 1e8
    else:
        do = do * (10.0 ** torch.linspace(-6, 0, Lq, device="cuda"))[None, None, :, None]
        v = v * (10.0 ** torch.linspace(-4, 0, Lk, device="cuda"))[None, None, :, None]
    ref = reference(q, k, v, do, None if bias is None else bias.expand(B, H, Lk))
    for name, a, b in zip(("out", "dq", "dk", "dv"), both(q, k, v, do, bias), ref):
        near(a, b, name)


def test_long():
    """Many tiles per accumulator: the error does not grow with the length."""
    q, do = randn(1, 1, 1, 4100, 64), randn(2, 1, 1, 4100, 64, scale=1e-3)
    k, v = randn(3, 1, 1, 4500, 64), randn(4, 1, 1, 4500, 64)
    for name, a, b in zip(("out", "dq", "dk", "dv"), both(q, k, v, do), reference(q, k, v, do)):
        near(a, b, name)


def test_differences():
    """<gradient, direction> against central differences of the forward kernel: a step of 2^-5 leaves its
    square times a third derivative of order one, fp32 rounding 1e-6 of the value over the step: 4e-3
    of the derivative's scale covers both."""
    import train_ops

    B, H, Lq, Lk = 1, 2, 37, 90
    t = {"q": randn(1, B, H, Lq, 64), "k": randn(2, B, H, Lk, 64), "v": randn(3, B, H, Lk, 64), "key_bias": randn(4, Lk)}
    do = randn(5, B, H, Lq, 64)
    grads = dict(zip(("q", "k", "v", "key_bias"), both(t["q"], t["k"], t["v"], do, t["key_bias"])[1:]))
    for i, name in enumerate(t):
        d = randn(10 + i, *t[name].shape)
        side = []
        for sign in (1, -1):
            x = dict(t, **{name: t[name] + sign * 2.0 ** -5 * d})
            side.append((train_ops.attention_forward(x["q"], x["k"], x["v"], key_bias=x["key_bias"])[0].double() * do.double()).sum().item())
        told = (grads[name].double() * d.double()).sum().item()
        scale = grads[name].double().norm().item() * d.double().norm().item()
        assert abs((side[0] - side[1]) * 2.0 ** 4 - told) <= 4e-3 * scale, name


def test_layouts_and_given_outputs():
    """Unaligned rows and every order of dimensions give the same bits; gradients into slices."""
    import train_ops

    B, H, Lq, Lk = 2, 3, 77, 141
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    first = both(q, k, v, do)

    def odd(t):  # rows 65 elements apart
        w = torch.zeros(*t.shape[:3], 65, device="cuda")
        w[..., 1:] = t
        return w[..., 1:]

    def swapped(t):
        return t.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)

    for turn in (odd, swapped, lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)):
        for a, b in zip(first[:4], both(*map(turn, (q, k, v, do)))[:4]):
            assert torch.equal(a, b)
    packed = torch.zeros(B, Lk, 3, H, 64, device="cuda")
    dq = odd(torch.zeros(B, H, Lq, 64, device="cuda"))
    grads = (dq, packed[:, :, 1].transpose(1, 2), packed[:, :, 2].transpose(1, 2))
    out, stats = train_ops.attention_forward(q, k, v)
    train_ops.attention_backward(do, q, k, v, out, stats, grads=grads)
    for a, b in zip(first[1:4], grads):
        assert torch.equal(a, b)
    assert not packed[:, :, 0].any()
    # a head of keys shared by all heads, expanded
    shared = k[:, :1].expand(B, H, Lk, 64), v[:, :1].expand(B, H, Lk, 64)
    for a, b in zip(both(q, *shared, do)[:4], both(q, *(t.contiguous() for t in shared), do)[:4]):
        assert torch.equal(a, b)


def test_forward_agrees_with_the_sampler_s_attention():
    """The inference entry on the same tensors: the same kernel, other scales of the split."""
    from native_sdpa_ctypes import native_sdpa_f32

    import train_ops

    q, k, v = (randn(i, 1, 2, 200, 64) for i in range(3))
    bias = randn(7, 200)
    near(train_ops.attention_forward(q, k, v, key_bias=bias)[0], native_sdpa_f32(q, k, v, key_bias=bias).double())


def test_side_stream_and_repeats():
    q, do, k, v = (randn(i, 2, 4, n, 64) for i, n in ((1, 500), (2, 500), (3, 700), (4, 700)))
    bias = randn(5, 700)
    first = both(q, k, v, do, bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = both(q, k, v, do, bias)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_refusals():
    import train_ops

    f = train_ops.attention_forward
    q, k = randn(1, 2, 2, 5, 64), randn(2, 2, 2, 7, 64)
    for call in (lambda: f(q[0], k, k), lambda: f(q[..., :32], k[..., :32], k[..., :32]), lambda: f(q.half(), k.half(), k.half()),
                 lambda: f(q, k, k[:, :, :5]), lambda: f(q, k[:, :1], k[:, :1]), lambda: f(q.cpu(), k.cpu(), k.cpu()),
                 lambda: f(q, k[:, :, :0], k[:, :, :0]), lambda: f(q, k, k, key_bias=torch.zeros(5, device="cuda")),
                 lambda: f(q, k, k, key_bias=torch.zeros(7)), lambda: f(q, k, k, key_bias=torch.zeros(7, device="cuda").half())):
        with pytest.raises(ValueError):
            call()
    out, stats = f(q, k, k)
    b = train_ops.attention_backward
    for call in (lambda: b(k, q, k, k, out, stats), lambda: b(q, q, k, k, out, stats[..., :1]),
                 lambda: b(q, q, k, k, out, stats, grads=(q, k)), lambda: b(q, q, k, k, out.half(), stats),
                 lambda: b(q, q, k, k, out, stats, grads=(q, k, k[:, :1].expand(2, 2, 7, 64)))):
        with pytest.raises(ValueError):
            call()
