"""Attention for training on both sides of the line between its two ways: few pairs of a query and a key (rows in
groups of four, fp32) and short sequences of so many heads that the tensor cores take them.  Definition in 64 bits;
tolerances and reference of test_attention_backward_gpu."""
import math

import pytest
import torch

from test_attention_backward_gpu import both, near, randn, reference

pytestmark = pytest.mark.gpu

NAMES = ("out", "dq", "dk", "dv")
FEW = [(1, 1, 5, 2), (1, 2, 6, 7), (2, 2, 65, 17), (1, 3, 9, 130), (1, 1, 130, 9), (1, 2, 100, 100), (1, 1, 7, 3000), (1, 1, 1000, 6)]
MANY = [(8, 16, 65, 17), (8, 32, 9, 40), (4, 32, 5, 1100), (8, 32, 700, 2), (16, 32, 40, 40), (2, 32, 127, 129), (16, 64, 16, 16),
        (4, 64, 64, 64), (8, 64, 33, 31)]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("size", FEW + MANY, ids=str)
def test_sizes(size, masked):
    B, H, Lq, Lk = size
    kv = randn(1, B, Lk, 2, H, 64)
    q, k, v = randn(2, B, Lq, H, 64).transpose(1, 2), kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    do = randn(3, B, Lq, H, 64).transpose(1, 2)
    bias = None
    if masked:  # the last request's first half missing; nothing missing elsewhere
        bias = randn(4, B, Lk)
        bias[-1, :Lk // 2] = -math.inf
    wide = None if bias is None else bias[:, None].expand(B, H, Lk)
    ref = reference(q, k, v, do, wide)
    out, dq, dk, dv, db = both(q, k, v, do, bias)
    # two keys, one of them missing, leave one: ds cancels to rounding there (floors as in test_sizes for one key)
    one = Lk == 2 and masked
    floor = (do.double().norm(dim=-1).mean() * v.double().norm(dim=-1).mean() / 64).item() if one else 0.0
    floors = {"dq": floor, "dk": floor * math.sqrt(Lq)}
    for name, a, b in zip(NAMES, (out, dq, dk, dv), ref):
        near(a, b, name, floors.get(name, 0.0))
    if masked:
        level = max(ref[4].square().sum((1, 2)).mean().sqrt().item(), floor * 64 * math.sqrt(H * Lq))
        near(db, ref[4].sum((1, 2)), "dbias", level)


def test_given_outputs_and_repeats():
    """Gradients into slices of a packed one, off the 16-byte boundaries; the same bits on every run."""
    B, H, Lq, Lk = 2, 3, 21, 50
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    first = both(q, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(first[:4], both(q, k, v, do)[:4]))
    buf = torch.full((B, Lk, H, 2 * 64 + 2), math.nan, device="cuda")
    dk, dv = buf[..., 1:65].transpose(1, 2), buf[..., 65:129].transpose(1, 2)
    dq = torch.empty(B, H, Lq, 65, device="cuda")[..., 1:]
    both(q, k, v, do, grads=(dq, dk, dv))
    assert torch.equal(dq, first[1]) and torch.equal(dk, first[2]) and torch.equal(dv, first[3])
    assert buf[..., 0].isnan().all() and buf[..., 129].isnan().all()


def test_both_ways_agree():
    """The same heads alone (few pairs) and among many."""
    H, Lq, Lk = 64, 40, 70
    q, do, k, v = (randn(i, 1, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    many = both(q, k, v, do)
    alone = both(q[:, :2], k[:, :2], v[:, :2], do[:, :2])
    for name, a, b in zip(NAMES, alone, many):
        near(a, b[:, :2].double(), name)
