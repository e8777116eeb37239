"""Operators for training on the flow model: attention with its backward pass, rotary positions
with several axes (and the per-head norm behind them), norms fused with a block's gate and
residual, gradient norm and clipping.

Each is a plain function on CUDA tensors, forward and backward apart, on PyTorch's current
stream; ``finetune.py`` puts them behind autograd and runs them together.  Arguments are
checked here (ValueError); a non-zero status of the library is a RuntimeError.  Tensors need a
contiguous last dimension and may have any strides otherwise (slices of a packed projection,
transposed heads); outputs are contiguous unless said otherwise.
"""
from __future__ import annotations

import struct

import torch

import _native

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_LAYOUTS = {"interleaved": 0, "halves": 1}
_KINDS = {None: 0, "layer": 1, "rms": 2}


_loaded = None


def _lib(device):
    """The library, with PyTorch's current stream set for its next launches."""
    global _loaded
    if device.type != "cuda":
        raise ValueError(f"expected CUDA tensors, got {device}")
    if device.index is not None and device.index != torch.cuda.current_device():
        raise ValueError(f"expected tensors on the current CUDA device, got {device}")
    if _loaded is None:
        _loaded = _native.load()
    _native.use_current_stream(_loaded)
    return _loaded


def _ok(lib, status, name):
    if status != 0:
        raise RuntimeError(f"{name} returned status {status}: {lib.triposplat_b200_last_error().decode()}")


def _check(t, name, shape, dtype, device):
    """`t` as a tensor of this shape, type and device (no conversion)."""
    if t.dtype is dtype and t.shape == shape and t.device == device:
        return t
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _param(t, name, shape, device):
    """A float32 parameter, contiguous; None stays None."""
    return None if t is None else _check(t, name, shape, torch.float32, device).contiguous()


def _rows(t):
    """`t` itself if its last dimension is contiguous, a contiguous copy otherwise."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


# Host arrays of the C interface, as bytes: a small call spends most of its time in Python, and
# packing takes a third of what filling a ctypes array does.
_I64 = [struct.Struct(f"{n}q") for n in range(33)]


def _i64(values):
    return _I64[len(values)].pack(*values)


def _strides(n, *tensors):
    """The first n strides of each tensor (zeros for None)."""
    values = []
    for t in tensors:
        values += (0,) * n if t is None else t.stride()[:n]
    return _i64(values)


# ------------------------------------------------------------------------ rotary positions
def _rope_args(x, positions, inv_freq, axis_pairs, gamma, layout):
    if x.dim() != 4 or x.dtype not in _DTYPES:
        raise ValueError("x must be [B, L, H, D] in float32, bfloat16 or float16")
    B, L, H, D = x.shape
    if min(B, L, H, D) < 1 or D % 2 or D > 256 or B > 65535:
        raise ValueError(f"unsupported shape {tuple(x.shape)}: no empty dimension, D even and up to 256")
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be 'interleaved' or 'halves', got {layout!r}")
    pairs = [int(p) for p in axis_pairs]
    if not 1 <= len(pairs) <= 4 or min(pairs) < 0 or sum(pairs) > D // 2:
        raise ValueError(f"axis_pairs {pairs} must be 1 to 4 counts of at most {D // 2} pairs in all")
    if positions.dtype not in _POSITIONS:
        raise ValueError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    if tuple(positions.shape) not in ((L, len(pairs)), (B, L, len(pairs))):
        raise ValueError(f"positions must be [L, axes] or [B, L, axes], got {tuple(positions.shape)}")
    if positions.device != x.device:
        raise ValueError(f"positions must be on {x.device}")
    inv_freq = _param(inv_freq, "inv_freq", (sum(pairs),), x.device)
    gamma = _param(gamma, "gamma", (H, D), x.device)
    positions = positions.contiguous()
    how = (_DTYPES[x.dtype], _POSITIONS[positions.dtype], L * len(pairs) if positions.dim() == 3 else 0,
           B, L, H, D, struct.pack(f"{len(pairs)}i", *pairs), len(pairs), _LAYOUTS[layout])
    return positions, inv_freq, gamma, how


def _out_like(out, x, name):
    """An output of x's shape and type: `out` if given (unit last stride), a new one otherwise."""
    if out is None:
        return x.new_empty(x.shape)
    _check(out, name, x.shape, x.dtype, x.device)
    if out.stride(-1) != 1 and out.shape[-1] != 1:
        raise ValueError(f"{name} needs a contiguous last dimension")
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError(f"{name} must not be expanded")
    return out


def axis_rope(x, positions, inv_freq, *, axis_pairs, gamma=None, layout="interleaved", out=None):
    """Rotates x [B, L, H, D] by its tokens' positions [L, axes] (or [B, L, axes]).

    The first sum(axis_pairs) pairs of each head turn, axis_pairs[a] of them by axis a's
    position times their entry of ``inv_freq``; a pair is elements (2p, 2p+1) ("interleaved")
    or (p, P+p) ("halves").  With ``gamma`` [H, D] the rotated vector r becomes
    r * sqrt(D) / max(|r|, 1e-12) * gamma.  ``out`` may be x itself."""
    positions, inv_freq, gamma, how = _rope_args(x, positions, inv_freq, axis_pairs, gamma, layout)
    x = _rows(x)
    y = _out_like(out, x, "out")
    lib = _lib(x.device)
    _ok(lib, lib.triposplat_b200_axis_rope(
        x.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), _ptr(gamma), y.data_ptr(),
        _strides(3, x, y), *how), "axis_rope")
    return y


def axis_rope_backward(dy, x, positions, inv_freq, *, axis_pairs, gamma=None, layout="interleaved",
                       out=None):
    """Gradients (dx, dgamma) of ``axis_rope`` at x (read only with ``gamma``; dgamma is None
    without).  ``out`` receives dx and may be dy itself."""
    positions, inv_freq, gamma, how = _rope_args(dy, positions, inv_freq, axis_pairs, gamma, layout)
    dy = _rows(dy)
    if gamma is not None:
        x = _rows(_check(x, "x", dy.shape, dy.dtype, dy.device))
    dx = _out_like(out, dy, "out")
    dgamma = None if gamma is None else torch.empty_like(gamma)
    lib = _lib(dy.device)
    _ok(lib, lib.triposplat_b200_axis_rope_backward(
        dy.data_ptr(), x.data_ptr() if gamma is not None else None, positions.data_ptr(),
        inv_freq.data_ptr(), _ptr(gamma), dx.data_ptr(), _ptr(dgamma),
        _strides(3, dy, x if gamma is not None else None, dx), *how), "axis_rope_backward")
    return dx, dgamma


# ------------------------------------------------------------- norms with gate and residual
def _norm_args(x, y, gate, scale, shift, pre, pre_weight, post, post_weight):
    if x.dim() != 3 or x.dtype not in _DTYPES:
        raise ValueError("x must be [B, L, C] in float32, bfloat16 or float16")
    B, L, C = x.shape
    if min(B, L, C) < 1 or C > 8192 or B > 65535:
        raise ValueError(f"unsupported shape {tuple(x.shape)}: no empty dimension, C up to 8192")
    if pre not in _KINDS or post not in _KINDS:
        raise ValueError("pre and post must be 'layer', 'rms' or None")
    if (scale is None) != (shift is None):
        raise ValueError("scale and shift come together")
    if pre is None and (scale is not None or pre_weight is not None):
        raise ValueError("scale, shift and pre_weight need a pre norm")
    if post is None and post_weight is not None:
        raise ValueError("post_weight needs a post norm")
    d = x.device
    _check(y, "y", x.shape, x.dtype, d)
    return (_param(gate, "gate", (B, C), d), _param(scale, "scale", (B, C), d), _param(shift, "shift", (B, C), d),
            _param(pre_weight, "pre_weight", (C,), d), _param(post_weight, "post_weight", (C,), d))


def norm_gate(x, y, *, gate=None, scale=None, shift=None, pre="layer", pre_weight=None, post=None,
              post_weight=None, residual_scale=1.0, eps=1e-6):
    """The end of one block and the start of the next, on x, y [B, L, C]:

        z = x + residual_scale * gate[b] * post_weight * post(y)
        h = pre_weight * pre(z) * (1 + scale[b]) + shift[b]

    post and pre are 'layer', 'rms' or None (no norm; without ``pre`` h is None); gate, scale and
    shift are [B, C], the weights [C], all float32 and optional.  Returns (z, h, stats); stats
    [B, L, 4] goes to the backward pass."""
    gate, scale, shift, wpre, wpost = _norm_args(x, y, gate, scale, shift, pre, pre_weight, post, post_weight)
    x, y = _rows(x), _rows(y)
    B, L, C = x.shape
    z = x.new_empty((B, L, C))
    h = x.new_empty((B, L, C)) if pre is not None else None
    stats = x.new_empty((B, L, 4), dtype=torch.float32)
    lib = _lib(x.device)
    _ok(lib, lib.triposplat_b200_norm_gate(
        x.data_ptr(), y.data_ptr(), _strides(2, x, y), _ptr(gate), _ptr(scale), _ptr(shift),
        _ptr(wpre), _ptr(wpost), z.data_ptr(), _ptr(h), stats.data_ptr(), _DTYPES[x.dtype], B, L, C, _KINDS[pre],
        _KINDS[post], float(residual_scale), float(eps)), "norm_gate")
    return z, h, stats


def norm_gate_backward(dz, dh, x, y, stats, *, gate=None, scale=None, shift=None, pre="layer",
                       pre_weight=None, post=None, post_weight=None, residual_scale=1.0, eps=1e-6):
    """Gradients of ``norm_gate`` from those of z and h (either may be None), as a dict with x, y
    and, for each that was given, gate, scale, shift, pre_weight and post_weight (else None)."""
    gate, scale, shift, wpre, wpost = _norm_args(x, y, gate, scale, shift, pre, pre_weight, post, post_weight)
    if dz is None and dh is None:
        raise ValueError("at least one of dz and dh is needed")
    if dh is not None and pre is None:
        raise ValueError("dh needs a pre norm")
    dz, dh = (None if t is None else _rows(_check(t, n, x.shape, x.dtype, x.device))
              for t, n in ((dz, "dz"), (dh, "dh")))
    x, y = _rows(x), _rows(y)
    B, L, C = x.shape
    stats = _check(stats, "stats", (B, L, 4), torch.float32, x.device).contiguous()
    g = {"x": x.new_empty((B, L, C)), "y": x.new_empty((B, L, C))}
    for name, t in (("gate", gate), ("scale", scale), ("shift", shift), ("pre_weight", wpre),
                    ("post_weight", wpost)):
        g[name] = None if t is None else torch.empty_like(t)
    lib = _lib(x.device)
    _ok(lib, lib.triposplat_b200_norm_gate_backward(
        _ptr(dz), _ptr(dh), x.data_ptr(), y.data_ptr(), _strides(2, x, y, dz, dh), stats.data_ptr(), _ptr(gate), _ptr(scale),
        _ptr(wpre), _ptr(wpost), g["x"].data_ptr(), g["y"].data_ptr(), _ptr(g["gate"]), _ptr(g["scale"]),
        _ptr(g["shift"]), _ptr(g["pre_weight"]), _ptr(g["post_weight"]), _DTYPES[x.dtype], B, L, C, _KINDS[pre],
        _KINDS[post], float(residual_scale)), "norm_gate_backward")
    return g


# --------------------------------------------------------------------------------- attention
def _attention_args(q, k, v, key_bias):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v must be [B, H, L, 64]")
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    if D != 64 or min(B, H, Lq, Lk) < 1:
        raise ValueError(f"unsupported shapes {tuple(q.shape)}, {tuple(k.shape)}: head_dim 64, no empty dimension")
    _check(q, "q", (B, H, Lq, 64), torch.float32, q.device)
    _check(k, "k", (B, H, Lk, 64), torch.float32, q.device)
    _check(v, "v", (B, H, Lk, 64), torch.float32, q.device)
    bias_dims = (1, 1)
    if key_bias is not None:
        shape = tuple(key_bias.shape)
        if shape not in ((Lk,), (B, Lk), (B, H, Lk)):
            raise ValueError(f"key_bias must be [Lk], [B, Lk] or [B, H, Lk], got {shape}")
        key_bias = _param(key_bias, "key_bias", shape, q.device)
        bias_dims = ((1, 1), (B, 1), (B, H))[len(shape) - 1]
    return key_bias, bias_dims, (B, H, Lq, Lk)


def attention_forward(q, k, v, *, key_bias=None):
    """softmax(q k^T / 8 + key_bias) v on q [B, H, Lq, 64] and k, v [B, H, Lk, 64] (float32), key_bias
    [Lk], [B, Lk] or [B, H, Lk].  A key with a bias of -inf does not exist; a query without keys
    gives zeros.  Returns (out, stats): out [B, H, Lq, 64] in token-major storage
    ([B, Lq, H, 64], what the out-projection reads), stats [B, H, Lq + 1, 2] for the backward pass.
    Heads shared by several queries' heads are passed expanded."""
    key_bias, bias_dims, (B, H, Lq, Lk) = _attention_args(q, k, v, key_bias)
    q, k, v = _rows(q), _rows(k), _rows(v)
    out = q.new_empty((B, Lq, H, 64))
    stats = q.new_empty((B, H, Lq + 1, 2))
    lib = _lib(q.device)
    _ok(lib, lib.triposplat_b200_attention_forward(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _strides(3, q, k, v),
        _ptr(key_bias), *bias_dims, out.data_ptr(), stats.data_ptr(), B, H, Lq, Lk), "attention_forward")
    return out.transpose(1, 2), stats


def attention_backward(dout, q, k, v, out, stats, *, key_bias=None, grads=None, bias_grad=True):
    """Gradients (dq, dk, dv, dbias) of ``attention_forward`` with the incoming dout [B, H, Lq, 64].

    ``grads`` may name the three tensors to write (e.g. slices of a packed gradient); otherwise they
    are new, in token-major storage.  dbias has key_bias's shape (None without a bias or with
    ``bias_grad=False``)."""
    key_bias, bias_dims, (B, H, Lq, Lk) = _attention_args(q, k, v, key_bias)
    dev = q.device
    dout = _rows(_check(dout, "dout", q.shape, torch.float32, dev))
    out = _rows(_check(out, "out", q.shape, torch.float32, dev))
    stats = _check(stats, "stats", (B, H, Lq + 1, 2), torch.float32, dev).contiguous()
    q, k, v = _rows(q), _rows(k), _rows(v)
    if grads is None:
        dq, dk, dv = (q.new_empty((B, n, H, 64)).transpose(1, 2) for n in (Lq, Lk, Lk))
    else:
        dq, dk, dv = (_out_like(g, like, "grads") for g, like in zip(grads, (q, k, v), strict=True))
    dbias = torch.empty_like(key_bias) if key_bias is not None and bias_grad else None
    lib = _lib(dev)
    _ok(lib, lib.triposplat_b200_attention_backward(
        dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), stats.data_ptr(),
        _strides(3, dout, q, k, v, out, dq, dk, dv), _ptr(key_bias), *bias_dims,
        dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dbias), B, H, Lq, Lk), "attention_backward")
    return dq, dk, dv, dbias


# -------------------------------------------------------------------- gradient norm, clipping
def clip_grad_norm(grads, max_norm, *, out=None):
    """Scales the gradients (a sequence of contiguous tensors, float32, bfloat16 and float16
    mixed as they come) by min(1, max_norm / (norm + 1e-6)), norm being their joint 2-norm; in
    place, or into the tensors of ``out``.  Returns the norm before clipping, a float32 scalar on
    the device; nothing waits for it.  A norm that is not finite scales as the formula says
    (NaN everywhere, or by zero)."""
    grads = list(grads)
    outs = grads if out is None else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"{len(grads)} gradients and {len(outs)} outputs")
    if not grads:
        raise ValueError("no gradients")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be zero or more, got {max_norm}")
    device, n = grads[0].device, len(grads)
    for g, o in zip(grads, outs):
        if g.device != device or o.device != device or g.dtype not in _DTYPES or o.dtype != g.dtype:
            raise ValueError("gradients and outputs must be float32, bfloat16 or float16 tensors of one device, "
                             "an output of its gradient's type")
        if not g.is_contiguous() or not o.is_contiguous() or o.shape != g.shape:
            raise ValueError("gradients and outputs must be contiguous, an output of its gradient's shape")
    norm = torch.empty((), dtype=torch.float32, device=device)
    lib = _lib(device)
    array = f"{n}q"
    ptrs = struct.pack(array, *[g.data_ptr() for g in grads])
    to = None if out is None else struct.pack(array, *[o.data_ptr() for o in outs])
    _ok(lib, lib.triposplat_b200_clip_grad_norm(
        ptrs, to, struct.pack(array, *[g.numel() for g in grads]),
        struct.pack(f"{n}i", *[_DTYPES[g.dtype] for g in grads]), n, max_norm, norm.data_ptr()), "clip_grad_norm")
    return norm
