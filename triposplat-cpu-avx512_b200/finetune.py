"""Training what is not quantised of the flow model's self-attention, with its NF24 Linears frozen.

The operators of ``train_ops`` behind autograd, and a small path that runs them together as a
training step does: ``AttentionTuner`` takes a model's weights (``flow_model.FlowWeights``), embeds
noisy latents, runs every block's self-attention (norm + modulation -> QKV Linear -> rotary positions
and per-head norm -> attention -> out Linear -> post norm, gate, residual), and predicts the
velocity; its parameters are the blocks' adaLN tables, per-head gains and post-norm weights.
``train_step`` adds the flow-matching loss, the backward pass, clipping and the update.

    python triposplat-cpu-avx512_b200/finetune.py --steps 30
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

import _native
import train_ops
from flow_model import FlowSpec, FlowWeights, make_weights, timestep_frequencies
from nf24_linear import nf24_linear


class _Attention(torch.autograd.Function):
    """Rotary positions and per-head norm on the query and key part of a packed projection
    [B, L, 3, H, 64], then attention; the gradient comes back packed, without copies."""

    @staticmethod
    def forward(ctx, qkv, gamma, positions, inv_freq, axis_pairs, key_bias):
        B, L, _, H, _ = qkv.shape
        qkv = qkv.contiguous()
        qk = train_ops.axis_rope(qkv.view(B, L, 3 * H, 64)[:, :, :2 * H], positions, inv_freq,
                                 axis_pairs=axis_pairs, gamma=gamma)
        q, k, v = (t.transpose(1, 2) for t in (qk[:, :, :H], qk[:, :, H:], qkv[:, :, 2]))
        out, stats = train_ops.attention_forward(q, k, v, key_bias=key_bias)
        ctx.save_for_backward(qkv, gamma, positions, inv_freq, key_bias, qk, out, stats)
        ctx.axis_pairs = axis_pairs
        return out.transpose(1, 2)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, gamma, positions, inv_freq, key_bias, qk, out, stats = ctx.saved_tensors
        B, L, _, H, _ = qkv.shape
        dqkv, dqk = torch.empty_like(qkv), torch.empty_like(qk)
        q, k, v, dq, dk, dv = (t.transpose(1, 2) for t in (qk[:, :, :H], qk[:, :, H:], qkv[:, :, 2], dqk[:, :, :H],
                                                           dqk[:, :, H:], dqkv[:, :, 2]))
        _, _, _, dbias = train_ops.attention_backward(
            dout.transpose(1, 2), q, k, v, out, stats, key_bias=key_bias, grads=(dq, dk, dv),
            bias_grad=ctx.needs_input_grad[5])
        _, dgamma = train_ops.axis_rope_backward(
            dqk, qkv.view(B, L, 3 * H, 64)[:, :, :2 * H], positions, inv_freq, axis_pairs=ctx.axis_pairs, gamma=gamma,
            out=dqkv.view(B, L, 3 * H, 64)[:, :, :2 * H])
        return dqkv, dgamma, None, None, None, dbias


class _NormGate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, scale, shift, pre_weight, post_weight, how):
        z, h, stats = train_ops.norm_gate(x, y, gate=gate, scale=scale, shift=shift, pre_weight=pre_weight,
                                          post_weight=post_weight, **how)
        ctx.save_for_backward(x, y, stats, gate, scale, shift, pre_weight, post_weight)
        ctx.how = how
        ctx.set_materialize_grads(False)
        return z, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dz, dh):
        x, y, stats, gate, scale, shift, pre_weight, post_weight = ctx.saved_tensors
        if dz is None and dh is None:
            return (None,) * 8
        g = train_ops.norm_gate_backward(dz, dh, x, y, stats, gate=gate, scale=scale, shift=shift,
                                         pre_weight=pre_weight, post_weight=post_weight, **ctx.how)
        return (g["x"], g["y"], g["gate"], g["scale"], g["shift"], g["pre_weight"], g["post_weight"], None)


class _FrozenLinear(torch.autograd.Function):
    """x W + b with a frozen NF24 weight; dx = (dy * scale) codes^T runs on the transposed codes."""

    @staticmethod
    def forward(ctx, x, lin):
        ctx.lin = lin
        p = lin.packed
        return nf24_linear(x, p.code01, p.q2, p.scale, p.bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        lin = ctx.lin
        return nf24_linear(dy * lin.packed.scale, lin.code01_nk, lin.q2_nk, lin.ones, lin.zeros), None


class FrozenLinear:
    """An NF24 Linear of a ``FlowWeights`` with a gradient to its input (not to its weight)."""

    def __init__(self, packed):
        self.packed = packed
        K, N = (int(d) for d in packed.code01.shape)
        device = packed.code01.device
        self.code01_nk = torch.empty(N, K, dtype=torch.int16, device=device)
        self.q2_nk = torch.empty(N, K, dtype=torch.int8, device=device)
        lib = _native.load()
        _native.use_current_stream(lib)
        st = lib.triposplat_b200_nf24_codes_to_nk(packed.code01.data_ptr(), packed.q2.data_ptr(), K, N,
                                                  self.code01_nk.data_ptr(), self.q2_nk.data_ptr())
        if st != 0:
            raise RuntimeError(f"nf24_codes_to_nk returned status {st}")
        self.ones = torch.ones(K, device=device)
        self.zeros = torch.zeros(K, device=device)

    def __call__(self, x):
        return _FrozenLinear.apply(x, self)


def attention(qkv, gamma, positions, inv_freq, *, axis_pairs, key_bias=None):
    """``train_ops.axis_rope`` (gamma [2 H, 64]: queries', then keys' gains) and attention on a packed
    projection [B, L, 3, H, 64], differentiable in qkv, gamma and key_bias; [B, L, H, 64]."""
    return _Attention.apply(qkv, gamma, positions, inv_freq, tuple(axis_pairs), key_bias)


def norm_gate(x, y, *, gate=None, scale=None, shift=None, pre="layer", pre_weight=None, post=None,
              post_weight=None, residual_scale=1.0, eps=1e-6):
    """``train_ops.norm_gate`` behind autograd: (z, h)."""
    how = dict(pre=pre, post=post, residual_scale=residual_scale, eps=eps)
    return _NormGate.apply(x, y, gate, scale, shift, pre_weight, post_weight, how)


def grid_positions(spec: FlowSpec, device="cuda"):
    """[L, 3] int32 grid positions of the latent tokens; the camera token at the origin."""
    gx, gy, gz = spec.grid
    n = torch.arange(spec.latent_tokens)
    pos = torch.stack([n // (gy * gz), (n // gz) % gy, n % gz], 1)
    return torch.cat([pos, torch.zeros(1, 3, dtype=pos.dtype)]).to(torch.int32).to(device)


def inverse_frequencies(spec: FlowSpec, device="cuda"):
    return torch.cat([1.0 / spec.theta ** (torch.arange(p, dtype=torch.float64) / p)
                      for p in spec.rope_pairs]).float().to(device)


class AttentionTuner(torch.nn.Module):
    """The self-attention path of a flow model with trainable tables, gains and post-norm weights."""

    def __init__(self, weights: FlowWeights):
        super().__init__()
        self.spec = s = weights.spec
        self.weights = weights
        names = ["x_embedder", "camera_embedder", "t_fc1", "t_fc2", "adaLN", "final_adaLN"]
        self.plain = {n: weights.linears[n] for n in names}  # before the first parameter: no gradient
        self.linears = {n: FrozenLinear(weights.linears[n]) for i in range(s.blocks)
                        for n in (f"blocks.{i}.qkv", f"blocks.{i}.out")}
        self.linears["final_linear"] = FrozenLinear(weights.linears["final_linear"])
        device = weights.params["blocks.0.table"].device
        self.positions, self.inv_freq = grid_positions(s, device), inverse_frequencies(s, device)
        self.tfreqs = torch.from_numpy(timestep_frequencies(s)).to(device)
        P = torch.nn.Parameter
        prm = weights.params
        # rows shift, scale, gate of the block's attention
        self.tables = torch.nn.ParameterList([P(prm[f"blocks.{i}.table"][:3].clone()) for i in range(s.blocks)])
        self.gammas = torch.nn.ParameterList(
            [P(torch.cat([prm[f"blocks.{i}.q_gamma"], prm[f"blocks.{i}.k_gamma"]])) for i in range(s.blocks)])
        self.post = torch.nn.ParameterList([P(torch.ones(s.hidden, device=device)) for _ in range(s.blocks)])

    def _lin(self, name, x):
        p = self.plain[name]
        return nf24_linear(x, p.code01, p.q2, p.scale, p.bias)

    @torch.no_grad()
    def embed(self, latents, camera, t1000):
        """Token embeddings [B, L, hidden] and the shared modulation of all blocks [B, 6, hidden], of
        the last norm [B, 2, hidden]."""
        s = self.spec
        angle = t1000[:, None] * self.tfreqs
        t = torch.nn.functional.silu(self._lin("t_fc1", torch.cat([angle.cos(), angle.sin()], 1)))
        t = torch.nn.functional.silu(self._lin("t_fc2", t))
        x = torch.cat([self._lin("x_embedder", latents), self._lin("camera_embedder", camera)], 1)
        B = x.shape[0]
        return x, self._lin("adaLN", t).view(B, 6, s.hidden), self._lin("final_adaLN", t).view(B, 2, s.hidden)

    def forward(self, latents, camera, t1000):
        """Velocity of the latents [B, N, latent_dim]."""
        s = self.spec
        x, mod, final = self.embed(latents, camera, t1000)
        rows = [mod[:, :3] + table for table in self.tables]  # [B, 3, hidden] per block: shift, scale, gate
        after = [(r[:, 0], r[:, 1]) for r in rows[1:]] + [(final[:, 0], final[:, 1])]
        z, h = norm_gate(x, x, shift=rows[0][:, 0], scale=rows[0][:, 1], residual_scale=0.0, eps=s.eps)
        for i in range(s.blocks):
            qkv = self.linears[f"blocks.{i}.qkv"](h).view(*h.shape[:2], 3, s.heads, 64)
            o = attention(qkv, self.gammas[i], self.positions, self.inv_freq, axis_pairs=s.rope_pairs)
            y = self.linears[f"blocks.{i}.out"](o.reshape(*h.shape))
            # this block's post norm, gate and residual with the next one's norm and modulation
            z, h = norm_gate(z, y, gate=rows[i][:, 2], shift=after[i][0], scale=after[i][1], post="rms",
                             post_weight=self.post[i], eps=s.eps)
        return self.linears["final_linear"](h[:, :s.latent_tokens])


def flow_loss(model, latents, camera, noise, t):
    """Flow matching on the straight path: x_t = (1 - t) x + t noise, velocity noise - x."""
    w = t[:, None, None]
    v = model((1 - w) * latents + w * noise, camera, 1000.0 * t)
    return (v - (noise - latents)).square().mean()


def train_step(model, optimizer, batch, max_norm: float = 1.0):
    """One step: loss, gradients, clipping by their global norm, update.  Returns (loss, norm) on the
    device."""
    optimizer.zero_grad(set_to_none=True)
    loss = flow_loss(model, *batch)
    loss.backward()
    norm = train_ops.clip_grad_norm([p.grad for p in model.parameters() if p.grad is not None], max_norm)
    optimizer.step()
    return loss.detach(), norm


def synthetic_batch(spec: FlowSpec, batch: int, seed: int, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *shape: torch.randn(*shape, generator=g, device=device)  # noqa: E731
    return (r(batch, spec.latent_tokens, spec.latent_dim), r(batch, 1, spec.camera_dim),
            r(batch, spec.latent_tokens, spec.latent_dim), torch.rand(batch, generator=g, device=device))


def main(argv=None):
    import argparse

    ap = argparse.ArgumentParser(description="Tune a synthetic flow model's attention (random weights and data).")
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--full", action="store_true", help="full-size blocks (8193 tokens, hidden 1024) instead of small ones")
    ap.add_argument("--batch", type=int, default=2)
    ap.add_argument("--lr", type=float, default=3e-2)
    ap.add_argument("--max-norm", type=float, default=1.0)
    a = ap.parse_args(argv)
    spec = FlowSpec(blocks=a.blocks) if a.full else FlowSpec.small(blocks=a.blocks)
    model = AttentionTuner(make_weights(spec, seed=0, device="cuda"))
    optimizer = torch.optim.Adam(model.parameters(), lr=a.lr)
    data = synthetic_batch(spec, a.batch, 1)
    for i in range(a.steps):
        loss, norm = train_step(model, optimizer, data, a.max_norm)
        if i % max(1, a.steps // 10) == 0 or i == a.steps - 1:
            print(f"step {i}: loss {loss.item():.5f}, gradient norm {norm.item():.4f}")
    return loss.item()


if __name__ == "__main__":
    main()
