"""Attention for training where keys are missing at either end of a row, in whole tiles of 128 and in
parts of them: the walk leaves such tiles out.  Definition in 64 bits; tolerances and reference of
test_attention_backward_gpu."""
import math

import pytest
import torch

from test_attention_backward_gpu import both, near, randn, reference

pytestmark = pytest.mark.gpu

NAMES = ("out", "dq", "dk", "dv")


def compare(got, ref, gone, floors={}):
    """Queries that have keys and keys that exist against `ref`, the others zero (level and error are those of
    the elements that are anything; gone [B, H, Lk])."""
    q = ~gone.all(-1)[..., None].expand(got[0].shape[:3])
    for name, a, b, there in zip(NAMES, got, ref, (q, q, ~gone, ~gone)):
        assert not a[~there].any(), name
        if there.any():
            near(a[there], b[there], name, floors.get(name, 0.0))


@pytest.mark.parametrize("ranges", [[(0, 1), (0, 128)], [(0, 129), (640, 700)], [(699, 700), (0, 0)], [(130, 250), (256, 384)],
                                    [(0, 0), (0, 0)], [(0, 700), (383, 513)]], ids=str)
@pytest.mark.parametrize("Lq", [2, 70, 1000])
def test_ranges(Lq, ranges):
    """Keys [first, last) of each request (with a hole in the long ones); the rest holds NaN."""
    B, H, Lk = 2, 3, 700
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    bias = randn(5, B, Lk)
    at = torch.arange(Lk, device="cuda")
    for b, (first, last) in enumerate(ranges):
        bias[b, (at < first) | (at >= last) | ((at >= 200) & (at < 350) & (last - first > 500))] = -math.inf
    wide = bias[:, None].expand(B, H, Lk)
    gone = wide == -math.inf
    hole = gone[..., None]
    ref = reference(q, k, v, do, wide)
    got = both(q, k.masked_fill(hole, math.nan), v.masked_fill(hole, math.nan), do, bias)
    # with one key ds cancels to rounding: measured against the terms it cancels from, Lq of them in dk
    single = max(last - first for first, last in ranges) == 1
    floor = (do.double().norm(dim=-1).mean() * v.double().norm(dim=-1).mean() / 64).item() if single else 0.0
    compare(got, ref, gone, {"dq": floor, "dk": floor * math.sqrt(Lq)})
    level = max(ref[4].square().sum((1, 2)).mean().sqrt().item(), floor * 64 * math.sqrt(H * Lq))
    near(got[4], ref[4].sum((1, 2)), "dbias", level)


@pytest.mark.parametrize("shape", [(1, 1, 5, 3000), (1, 2, 3000, 300), (1, 1, 64, 8193)], ids=str)
def test_cut_walks(shape):
    """Shares of a walk that hold no key at all."""
    B, H, Lq, Lk = shape
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    bias = randn(5, B, H, Lk)
    bias[:, 0, Lk // 3:] = -math.inf
    bias[:, -1, :Lk // 4] = -math.inf
    ref = reference(q, k, v, do, bias)
    compare(both(q, k, v, do, bias), ref, bias == -math.inf)


def test_many_heads_of_different_length():
    """More work items than the GPU holds at a time, with empty ones between the others."""
    B, H, Lq, Lk = 9, 16, 200, 400
    q, do, k, v = (randn(i, B, H, n, 64) for i, n in ((1, Lq), (2, Lq), (3, Lk), (4, Lk)))
    bias = randn(5, B, H, Lk)
    ends = torch.randint(0, Lk + 1, (B, H, 1), generator=torch.Generator("cuda").manual_seed(6), device="cuda")
    ends[::2, ::3] = 0
    bias.masked_fill_(torch.arange(Lk, device="cuda") >= ends, -math.inf)
    ref = reference(q, k, v, do, bias)
    got = both(q, k, v, do, bias)
    compare(got, ref, bias == -math.inf)
    again = both(q, k, v, do, bias)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
