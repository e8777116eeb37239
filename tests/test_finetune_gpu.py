"""The training path as a whole: gradients of two blocks against the same computation in 64 bits on the
dequantised weights, and a few steps that lower the loss.

Tolerance.  The Linears, attention and norms are each within 2e-6 of their definition (2-norm); two
blocks chain some 30 of them forward and backward, so a gradient is within 30 * 2e-6 = 6e-5.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def linear(p, x):
    w = (p.code01.double() * 256 + p.q2.double()) * p.scale.double()
    return x @ w + p.bias.double()


def norm(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / (v.square().mean(-1, keepdim=True) + eps).sqrt()


def reference_loss(m, latents, camera, noise, t, tables, gammas, post):
    s, lin = m.spec, m.weights.linears
    d = lambda v: v.double()  # noqa: E731
    w = d(t)[:, None, None]
    xt = (1 - w) * d(latents) + w * d(noise)
    angle = 1000 * d(t)[:, None] * d(m.tfreqs)
    e = torch.nn.functional.silu(linear(lin["t_fc1"], torch.cat([angle.cos(), angle.sin()], 1)))
    e = torch.nn.functional.silu(linear(lin["t_fc2"], e))
    z = torch.cat([linear(lin["x_embedder"], xt), linear(lin["camera_embedder"], d(camera))], 1)
    B, L, C = z.shape
    mod, final = linear(lin["adaLN"], e).view(B, 6, C), linear(lin["final_adaLN"], e).view(B, 2, C)
    axis = [a for a, p in enumerate(s.rope_pairs) for _ in range(p)]
    turn = torch.exp(1j * d(m.positions)[:, axis] * d(m.inv_freq))[:, None]
    for i in range(s.blocks):
        r = (mod[:, :3] + tables[i])[:, :, None]
        h = norm(z, "layer", s.eps) * (1 + r[:, 1]) + r[:, 0]
        qkv = linear(lin[f"blocks.{i}.qkv"], h).view(B, L, 3, s.heads, 64)
        qk = qkv[:, :, :2].reshape(B, L, 2 * s.heads, 32, 2)
        qk = torch.view_as_real(torch.view_as_complex(qk.contiguous()) * turn).reshape(B, L, 2 * s.heads, 64)
        qk = qk * 8 / qk.norm(dim=-1, keepdim=True) * gammas[i]
        q, k, v = (x.transpose(1, 2) for x in (qk[:, :, :s.heads], qk[:, :, s.heads:], qkv[:, :, 2]))
        o = (q @ k.mT / 8).softmax(-1) @ v
        y = linear(lin[f"blocks.{i}.out"], o.transpose(1, 2).reshape(B, L, C))
        z = z + r[:, 2] * post[i] * norm(y, "rms", s.eps)
    h = norm(z, "layer", s.eps) * (1 + final[:, None, 1]) + final[:, None, 0]
    out = linear(lin["final_linear"], h[:, :s.latent_tokens])
    return (out - (d(noise) - d(latents))).square().mean()


@pytest.fixture(scope="module")
def tuner():
    import finetune
    from flow_model import FlowSpec, make_weights

    return finetune.AttentionTuner(make_weights(FlowSpec.small(blocks=2), seed=5, device="cuda"))


def test_gradients(tuner):
    import finetune

    batch = finetune.synthetic_batch(tuner.spec, 3, 2)
    groups = [[p.detach().double().requires_grad_() for p in g] for g in (tuner.tables, tuner.gammas, tuner.post)]
    ref = reference_loss(tuner, *batch, *groups)
    flat = [p for g in groups for p in g]
    ref_grads = torch.autograd.grad(ref, flat)
    loss = finetune.flow_loss(tuner, *batch)
    assert abs(loss.item() - ref.item()) <= 6e-5 * ref.item()
    grads = torch.autograd.grad(loss, [*tuner.tables, *tuner.gammas, *tuner.post])
    for i, (a, b) in enumerate(zip(grads, ref_grads)):
        assert (a.double() - b).norm().item() <= 6e-5 * b.norm().item(), i


def test_steps_lower_the_loss(tuner):
    import copy

    import finetune

    start = copy.deepcopy(tuner.state_dict())
    data = finetune.synthetic_batch(tuner.spec, 2, 7)
    optimizer = torch.optim.Adam(tuner.parameters(), lr=3e-2)
    first, norm = finetune.train_step(tuner, optimizer, data, max_norm=0.5)
    grads = [p.grad for p in tuner.parameters()]
    clipped = math.sqrt(sum(g.double().square().sum().item() for g in grads))
    assert clipped <= min(norm.item(), 0.5) * (1 + 1e-5)
    for _ in range(30):
        last, _ = finetune.train_step(tuner, optimizer, data, max_norm=0.5)
    assert last.item() < 0.98 * first.item(), (first.item(), last.item())
    tuner.load_state_dict(start)


def test_frozen_linear_input_gradient(tuner):
    """dx of an NF24 Linear against W^T in 64 bits, also for a width that is no multiple of 64."""
    import finetune

    for name in ("blocks.0.qkv", "blocks.1.out", "final_linear"):
        lin = tuner.linears[name]
        K, N = lin.packed.code01.shape
        x = torch.randn(5, 7, K, device="cuda", requires_grad=True)
        dy = torch.randn(5, 7, N, device="cuda")
        (dx,) = torch.autograd.grad(lin(x), x, dy)
        w = (lin.packed.code01.double() * 256 + lin.packed.q2.double()) * lin.packed.scale.double()
        ref = dy.double() @ w.T
        assert (dx.double() - ref).norm().item() <= 2e-6 * ref.norm().item(), name


def test_command(capsys):
    import finetune

    assert math.isfinite(finetune.main(["--steps", "3"]))
    assert "gradient norm" in capsys.readouterr().out
