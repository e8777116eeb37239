"""Attention for training where values leave the usual range: gradients near the ends of what fp32
holds, and infinities and NaN in single rows.  Definition in 64 bits; tolerances and reference of
test_attention_backward_gpu (what is finite has the same accuracy of scores and products)."""
import math

import pytest
import torch

from test_attention_backward_gpu import both, near, randn, reference

pytestmark = pytest.mark.gpu

NAMES = ("out", "dq", "dk", "dv")


def inputs(Lq, Lk):
    return [randn(i, 1, 2, n, 64) for i, n in ((1, Lq), (2, Lk), (3, Lk), (4, Lq))]


@pytest.mark.parametrize("scale", [1e-25, 1e18, 1e25])
@pytest.mark.parametrize("size", [(2, 70), (130, 200)], ids=str)
def test_far_gradients(size, scale):
    """The squares of such gradients are zero or infinite in 32 bits."""
    q, k, v, do = inputs(*size)
    do = do * scale
    for name, a, b in zip(NAMES, both(q, k, v, do), reference(q, k, v, do)):
        near(a, b, name)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("size", [(3, 70), (130, 200)], ids=str)
def test_a_row_of_the_gradient(size, bad):
    """dO of one query not finite: its dQ and its head's dK, and the others' dQ as if it were not there."""
    q, k, v, do = inputs(*size)
    ref = reference(q, k, v, do)
    do = do.clone()
    do[0, 0, 1, 5] = bad
    out, dq, dk, dv, _ = both(q, k, v, do)
    near(out, ref[0])
    assert not dq[0, 0, 1].isfinite().any() and not dk[0, 0].isfinite().any() and not dv[0, 0, :, 5].isfinite().any()
    near(dq[0, 0, 2:], ref[1][0, 0, 2:])
    near(dk[0, 1], ref[2][0, 1])
    for d in (slice(0, 5), slice(6, 64)):
        near(dv[0, 0, :, d], ref[3][0, 0, :, d])


@pytest.mark.parametrize("size", [(3, 70), (130, 200), (700, 300)], ids=str)
@pytest.mark.parametrize("what", ["q", "k", "v", "bias"])
def test_nothing_is_hidden(size, what):
    """A NaN reaches every element that depends on it, and a query's own NaN no other query."""
    Lq, Lk = size
    q, k, v, do = inputs(Lq, Lk)
    bias = randn(5, 1, 2, Lk)
    t = {"q": q, "k": k, "v": v, "bias": bias[..., None]}[what]
    ref = reference(q, k, v, do, bias)
    t[0, 0, 2, 0] = math.nan
    out, dq, dk, dv, db = both(q, k, v, do, bias)
    if what == "q":
        assert out[0, 0, 2].isnan().all() and dq[0, 0, 2].isnan().all()
        near(torch.cat([out[0, 0, :2], out[0, 0, 3:]]), torch.cat([ref[0][0, 0, :2], ref[0][0, 0, 3:]]))
        near(torch.cat([dq[0, 0, :2], dq[0, 0, 3:]]), torch.cat([ref[1][0, 0, :2], ref[1][0, 0, 3:]]))
    elif what == "v":
        assert out[0, 0, :, 0].isnan().all() and dq[0, 0].isnan().all()
        near(out[0, 0, :, 1:], ref[0][0, 0, :, 1:])
    else:
        assert out[0, 0].isnan().all() and dq[0, 0].isnan().all()
    assert dk[0, 0].isnan().all() and db[0, 0].isnan().all()
    assert dv[0, 0].isnan().all() if what != "v" else torch.isfinite(dv).all()
    for name, a, b in zip(NAMES, (out, dq, dk, dv), ref):
        near(a[0, 1], b[0, 1], name)
