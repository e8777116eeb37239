"""Operators for training on the flow model: attention with its backward pass, rotary positions
with several axes (and the per-head norm behind them), norms fused with a block's gate and
residual, gradient norm and clipping.

Each is a plain function on CUDA tensors, forward and backward apart, on PyTorch's current
stream; ``finetune.py`` puts them behind autograd and runs them together.  Arguments are
checked (ValueError); a non-zero status of the library is a RuntimeError.  Tensors need a
contiguous last dimension and may have any strides otherwise (slices of a packed projection,
transposed heads); outputs are contiguous unless said otherwise.
"""
from __future__ import annotations

import ctypes

import torch  # noqa: F401  (before train_calls, which is linked against it)

import _native
import train_calls

_LAYOUTS = {"interleaved": 0, "halves": 1}
_KINDS = {None: 0, "layer": 1, "rms": 2}

# train_calls.cpp's order
_FUNCTIONS = ("set_stream", "last_error", "axis_rope", "axis_rope_backward", "norm_gate", "norm_gate_backward",
              "attention_forward", "attention_backward", "clip_grad_norm")
_library = _native.load()
train_calls.bind([ctypes.cast(getattr(_library, "triposplat_b200_" + f), ctypes.c_void_p).value for f in _FUNCTIONS])


# ------------------------------------------------------------------------ rotary positions
def axis_rope(x, positions, inv_freq, *, axis_pairs, gamma=None, layout="interleaved", out=None):
    """Rotates x [B, L, H, D] by its tokens' positions [L, axes] (or [B, L, axes]).

    The first sum(axis_pairs) pairs of each head turn, axis_pairs[a] of them by axis a's
    position times their entry of ``inv_freq``; a pair is elements (2p, 2p+1) ("interleaved")
    or (p, P+p) ("halves").  With ``gamma`` [H, D] the rotated vector r becomes
    r * sqrt(D) / max(|r|, 1e-12) * gamma.  ``out`` may be x itself."""
    return train_calls.axis_rope(x, positions, inv_freq, axis_pairs, gamma, _LAYOUTS.get(layout, -1), out)


def axis_rope_backward(dy, x, positions, inv_freq, *, axis_pairs, gamma=None, layout="interleaved",
                       out=None):
    """Gradients (dx, dgamma) of ``axis_rope`` at x (read only with ``gamma``; dgamma is None
    without).  ``out`` receives dx and may be dy itself."""
    return train_calls.axis_rope_backward(dy, x, positions, inv_freq, axis_pairs, gamma, _LAYOUTS.get(layout, -1), out)


# ------------------------------------------------------------- norms with gate and residual
def norm_gate(x, y, *, gate=None, scale=None, shift=None, pre="layer", pre_weight=None, post=None,
              post_weight=None, residual_scale=1.0, eps=1e-6):
    """The end of one block and the start of the next, on x, y [B, L, C]:

        z = x + residual_scale * gate[b] * post_weight * post(y)
        h = pre_weight * pre(z) * (1 + scale[b]) + shift[b]

    post and pre are 'layer', 'rms' or None (no norm; without ``pre`` h is None); gate, scale and
    shift are [B, C], the weights [C], all float32 and optional.  Returns (z, h, stats); stats
    [B, L, 4] goes to the backward pass."""
    return train_calls.norm_gate(x, y, gate, scale, shift, _KINDS.get(pre, -1), pre_weight, _KINDS.get(post, -1),
                                 post_weight, residual_scale, eps)


def norm_gate_backward(dz, dh, x, y, stats, *, gate=None, scale=None, shift=None, pre="layer",
                       pre_weight=None, post=None, post_weight=None, residual_scale=1.0, eps=1e-6):
    """Gradients of ``norm_gate`` from those of z and h (either may be None), as a dict with x, y
    and, for each that was given, gate, scale, shift, pre_weight and post_weight (else None)."""
    dx, dy, dgate, dscale, dshift, dpre, dpost = train_calls.norm_gate_backward(
        dz, dh, x, y, stats, gate, scale, shift, _KINDS.get(pre, -1), pre_weight, _KINDS.get(post, -1), post_weight,
        residual_scale)
    return {"x": dx, "y": dy, "gate": dgate, "scale": dscale, "shift": dshift, "pre_weight": dpre,
            "post_weight": dpost}


# --------------------------------------------------------------------------------- attention
def attention_forward(q, k, v, *, key_bias=None):
    """softmax(q k^T / 8 + key_bias) v on q [B, H, Lq, 64] and k, v [B, H, Lk, 64] (float32), key_bias
    [Lk], [B, Lk] or [B, H, Lk].  A key with a bias of -inf does not exist; a query without keys
    gives zeros.  Returns (out, stats): out [B, H, Lq, 64] in token-major storage
    ([B, Lq, H, 64], what the out-projection reads), stats [B, H, Lq + 1, 2] for the backward pass.
    Heads shared by several queries' heads are passed expanded."""
    return train_calls.attention_forward(q, k, v, key_bias)


def attention_backward(dout, q, k, v, out, stats, *, key_bias=None, grads=None, bias_grad=True):
    """Gradients (dq, dk, dv, dbias) of ``attention_forward`` with the incoming dout [B, H, Lq, 64].

    ``grads`` may name the three tensors to write (e.g. slices of a packed gradient); otherwise they
    are new, in token-major storage.  dbias has key_bias's shape (None without a bias or with
    ``bias_grad=False``)."""
    return train_calls.attention_backward(dout, q, k, v, out, stats, key_bias, grads, bias_grad)


# -------------------------------------------------------------------- gradient norm, clipping
def clip_grad_norm(grads, max_norm, *, out=None):
    """Scales the gradients (a sequence of contiguous tensors, float32, bfloat16 and float16
    mixed as they come) by min(1, max_norm / (norm + 1e-6)), norm being their joint 2-norm; in
    place, or into the tensors of ``out``.  Returns the norm before clipping, a float32 scalar on
    the device; nothing waits for it.  A norm that is not finite scales as the formula says
    (NaN everywhere, or by zero)."""
    return train_calls.clip_grad_norm(grads, max_norm, out)
