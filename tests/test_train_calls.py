"""Refusals of the training operators' Python calls that need no device, and the calls' bookkeeping."""
import math

import pytest
import torch


@pytest.fixture(scope="module")
def ops():
    import build_lib

    build_lib.build()
    import train_ops

    return train_ops


X, POS, INV = torch.zeros(1, 4, 2, 64), torch.zeros(4, 1, dtype=torch.int32), torch.ones(32)


@pytest.mark.parametrize("change, words", [
    (dict(x=X[0]), "x must be"), (dict(x=X.double()), "x must be"), (dict(x=X[..., :63]), "unsupported shape"),
    (dict(x=X[:, :0]), "unsupported shape"), (dict(axis_pairs=[33]), "axis_pairs"), (dict(axis_pairs=[]), "axis_pairs"),
    (dict(axis_pairs=[-1, 4]), "axis_pairs"), (dict(axis_pairs=[8] * 5), "axis_pairs"), (dict(layout="pairs"), "layout"),
    (dict(positions=POS.half()), "positions must be int32"), (dict(positions=POS[:3]), "positions must be \\[L"),
    (dict(inv_freq=INV[:31]), "inv_freq must have shape \\(32,\\), got \\(31,\\)"),
    (dict(inv_freq=INV.double()), "inv_freq must be torch.float32, got torch.float64"),
    (dict(gamma=torch.ones(2, 63)), "gamma must have shape"), (dict(out=X.half()), "out must be torch.float32"),
    (dict(out=X[:, :1].expand(1, 4, 2, 64)), "out must not be expanded"),
    (dict(out=torch.zeros(1, 4, 2, 128)[..., ::2]), "contiguous last"), (dict(), "expected CUDA tensors, got cpu")], ids=str)
def test_rope(ops, change, words):
    a = dict(x=X, positions=POS, inv_freq=INV, axis_pairs=[32]) | change
    with pytest.raises(ValueError, match=words):
        ops.axis_rope(a.pop("x"), a.pop("positions"), a.pop("inv_freq"), **a)


def test_norm(ops):
    t, w = torch.zeros(2, 3, 8), torch.ones(8)
    stats = torch.zeros(2, 3, 4)
    for call, words in ((lambda: ops.norm_gate(t, t[:1]), "y must have shape"), (lambda: ops.norm_gate(t, t, pre="batch"), "pre and post"),
                        (lambda: ops.norm_gate(t, t, scale=t[:, 0]), "together"),
                        (lambda: ops.norm_gate(t, t, pre=None, pre_weight=w), "need a pre norm"),
                        (lambda: ops.norm_gate(t, t, post_weight=w), "needs a post norm"),
                        (lambda: ops.norm_gate(t, t, gate=w), "gate must have shape"),
                        (lambda: ops.norm_gate_backward(None, None, t, t, stats), "at least one"),
                        (lambda: ops.norm_gate_backward(t, t, t, t, stats, pre=None), "dh needs"),
                        (lambda: ops.norm_gate_backward(t, t[:1], t, t, stats), "dh must have shape"),
                        (lambda: ops.norm_gate(t, t), "expected CUDA")):
        with pytest.raises(ValueError, match=words):
            call()


def test_attention(ops):
    q, k = torch.zeros(2, 2, 5, 64), torch.zeros(2, 2, 7, 64)
    stats = torch.zeros(2, 2, 6, 2)
    for call, words in ((lambda: ops.attention_forward(q[0], k, k), "must be \\[B, H, L, 64\\]"),
                        (lambda: ops.attention_forward(q[..., :32], k, k), "head_dim 64"),
                        (lambda: ops.attention_forward(q, k[:, :, :0], k), "no empty"),
                        (lambda: ops.attention_forward(q, k, k[:, :, :5]), "v must have shape"),
                        (lambda: ops.attention_forward(q, k, k, key_bias=torch.zeros(5)), "key_bias must be \\[Lk\\]"),
                        (lambda: ops.attention_backward(q, q, k, k, q, stats[..., :1]), "stats must have shape"),
                        (lambda: ops.attention_backward(q, q, k, k, q, stats, grads=(q, k)), "three tensors"),
                        (lambda: ops.attention_backward(q, q, k, k, q, stats, grads=(q, k, None)), "three tensors"),
                        (lambda: ops.attention_backward(q, q, k, k, q, stats, grads=(q, k, k[:, :, :1].expand(2, 2, 7, 64))), "expanded"),
                        (lambda: ops.attention_forward(q, k, k), "expected CUDA")):
        with pytest.raises(ValueError, match=words):
            call()


def test_clip(ops):
    t = torch.zeros(3, 4)
    for call, words in ((lambda: ops.clip_grad_norm([], 1.0), "no gradients"), (lambda: ops.clip_grad_norm([t], -1.0), "zero or more"),
                        (lambda: ops.clip_grad_norm([t], math.nan), "zero or more"), (lambda: ops.clip_grad_norm([t.double()], 1.0), "float32, bfloat16"),
                        (lambda: ops.clip_grad_norm([t[:, ::2]], 1.0), "contiguous"), (lambda: ops.clip_grad_norm([t], 1.0, out=[]), "1 gradients and 0"),
                        (lambda: ops.clip_grad_norm((g for g in [t, t]), 1.0), "expected CUDA")):
        with pytest.raises(ValueError, match=words):
            call()


def test_what_is_no_tensor_is_a_type_error(ops):
    """... and leaves the arguments' reference counts as they were."""
    import sys

    before = sys.getrefcount(X), sys.getrefcount(POS)
    for _ in range(50):
        for call in (lambda: ops.axis_rope(None, POS, INV, axis_pairs=[32]), lambda: ops.axis_rope(X, 3, INV, axis_pairs=[32]),
                     lambda: ops.axis_rope(X, POS, INV, axis_pairs=[3.5]), lambda: ops.axis_rope(X, POS, INV, axis_pairs=4),
                     lambda: ops.clip_grad_norm(4, 1.0), lambda: ops.clip_grad_norm([X], "1"),
                     lambda: ops.attention_forward(X, X, "x")):
            with pytest.raises(TypeError):
                call()
    assert (sys.getrefcount(X), sys.getrefcount(POS)) == before
