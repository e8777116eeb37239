"""Attention for training at the shapes that take ways of their own: up to four queries, and few
enough held rows that the walk over the other side is cut into shares.  Definition in 64 bits;
tolerances and reference of test_attention_backward_gpu (same accuracy of scores and products)."""
import math

import pytest
import torch

from test_attention_backward_gpu import both, near, randn, reference

pytestmark = pytest.mark.gpu

NAMES = ("out", "dq", "dk", "dv")


@pytest.mark.parametrize("Lk", [2, 63, 64, 65, 513, 3000])
@pytest.mark.parametrize("Lq", [1, 2, 3, 4])
def test_few_queries(Lq, Lk):
    B, H = 2, 3
    q, do = randn(1, B, Lq, H, 64).transpose(1, 2), randn(2, B, H, Lq, 64, scale=1e-3)
    kv = randn(3, B, Lk, 2, H, 64)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    for name, a, b in zip(NAMES, both(q, k, v, do), reference(q, k, v, do)):
        near(a, b, name)


@pytest.mark.parametrize("shape", [(1, 2, 5, 2000), (2, 1, 130, 3000), (1, 1, 64, 8193), (1, 2, 3000, 20), (1, 1, 4100, 129), (2, 2, 9, 777)], ids=str)
@pytest.mark.parametrize("masked", [False, True])
def test_cut_walks(shape, masked):
    B, H, Lq, Lk = shape
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    bias = wide = None
    if masked:
        bias = randn(5, B, Lk)
        bias[:, Lk // 3:Lk // 2] = -math.inf
        bias[-1, Lk // 4:] = -math.inf  # whole shares without a key
        wide = bias[:, None].expand(B, H, Lk)
    got, ref = both(q, k, v, do, bias), reference(q, k, v, do, wide)
    for name, a, b in zip(NAMES, got, ref):
        near(a, b, name)
    if masked:
        near(got[4], ref[4].sum((1, 2)), "dbias")


@pytest.mark.parametrize("Lq", [1, 3])
def test_few_queries_with_a_bias(Lq):
    """Missing keys that hold anything, a batch entry without keys, lowest values, shared and own rows."""
    B, H, Lk = 2, 2, 700
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    bias = randn(5, B, H, Lk)
    bias[torch.rand(B, H, Lk, device="cuda", generator=torch.Generator("cuda").manual_seed(6)) < 0.4] = -math.inf
    hole = bias == -math.inf
    ref = reference(q, k, v, do, bias)
    got = both(q, k.masked_fill(hole[..., None], math.nan), v.masked_fill(hole[..., None], math.inf), do, bias)
    for name, a, b in zip(NAMES, got, ref):
        near(a, b, name)
    near(got[4], ref[4].sum(2), "dbias")
    assert not got[2][hole].any() and not got[3][hole].any()
    shared = bias[0, 0]
    near(both(q, k, v, do, shared)[4], reference(q, k, v, do, shared.expand(B, H, Lk))[4].sum((0, 1, 2)), "dbias")
    none = torch.zeros(B, Lk, device="cuda")
    none[0] = -math.inf
    got = both(q, k, v, do, none)
    for t in got:
        assert not t[0].any() and torch.isfinite(t).all()
    low = torch.full((Lk,), torch.finfo(torch.float32).min, device="cuda")
    for a, b in zip(both(q, k, v, do, low)[:4], reference(q, k, v, do, torch.zeros(B, H, Lk, device="cuda"), scores=False)):
        near(a, b)


def test_few_queries_layouts_and_repeats():
    """The same bits from any strides, into given slices, and on every run."""
    import train_ops

    B, H, Lq, Lk = 2, 3, 3, 600
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    first = both(q, k, v, do)

    def odd(t):
        w = torch.zeros(*t.shape[:3], 67, device="cuda")
        w[..., 3:] = t
        return w[..., 3:]

    for a, b in zip(first[:4], both(*map(odd, (q, k, v, do)))[:4]):
        assert torch.equal(a, b)
    packed = odd(torch.zeros(B, H, 2 * Lk, 64, device="cuda"))
    grads = (odd(torch.zeros_like(q)), packed[:, :, :Lk], packed[:, :, Lk:])
    out, stats = train_ops.attention_forward(q, k, v)
    train_ops.attention_backward(do, q, k, v, out, stats, grads=grads)
    for a, b in zip(first[1:4], grads):
        assert torch.equal(a, b)
    long = randn(7, 1, 1, 40, 64), randn(8, 1, 1, 5000, 64), randn(9, 1, 1, 5000, 64), randn(10, 1, 1, 40, 64)
    assert all(torch.equal(a, b) for a, b in zip(both(*long)[:4], both(*long)[:4]))
