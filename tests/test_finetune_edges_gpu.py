"""Autograd's edges of the training path: second derivatives are refused, unused outputs and inputs
without a gradient take part as autograd means it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


def test_second_derivatives_are_refused():
    """The backward passes are kernels without a derivative of their own: an error, not a gradient that
    lacks their part."""
    import finetune

    x, y = (randn(i, 1, 5, 64).requires_grad_() for i in (1, 2))
    z, h = finetune.norm_gate(x, y, post="rms")
    g, = torch.autograd.grad(h.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    qkv = randn(3, 1, 5, 3, 2, 64).requires_grad_()
    pos, inv = torch.zeros(5, 1, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda")
    o = finetune.attention(qkv, torch.ones(4, 64, device="cuda"), pos, inv, axis_pairs=[32])
    g, = torch.autograd.grad(o.square().sum(), qkv, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_one_output_or_input_alone():
    import finetune

    x, y = randn(1, 2, 9, 64), randn(2, 2, 9, 64).requires_grad_()
    z, h = finetune.norm_gate(x, y, pre=None, post="layer")
    assert h is None
    z.sum().backward()  # an expanded gradient
    first, y.grad = y.grad, None
    ref = (y.double() - y.double().mean(-1, keepdim=True))
    ref = x.double() + ref / (ref.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    want, = torch.autograd.grad(ref.sum(), y)
    # sums of 64 terms of unit size that cancel: each within 64 roundings of 2^-24
    assert (first - want).abs().max() <= 64 * 64 * 2.0 ** -24
    z, h = finetune.norm_gate(x, y, post="layer")
    z.square().sum().backward()
    assert y.grad.isfinite().all() and x.grad is None
