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
    """`t` with a contiguous last dimension (a copy only if it has none), and its strides."""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] != 1:
        t = t.contiguous()
        st = t.stride()
    return t, st


def _ptr(t):
    return None if t is None else t.data_ptr()


# Host arrays of the C interface, as bytes: a small call spends most of its time in Python, and
# packing takes a third of what filling a ctypes array does.
_I64 = [struct.Struct(f"{n}q") for n in range(25)]


# ------------------------------------------------------------------------ rotary positions
def _rope_args(x, positions, inv_freq, axis_pairs, gamma, layout):
    code = _DTYPES.get(x.dtype)
    if x.dim() != 4 or code is None:
        raise ValueError("x must be [B, L, H, D] in float32, bfloat16 or float16")
    B, L, H, D = x.shape
    if D % 2 or not 0 < D <= 256 or not (B and L and H) or B > 65535:
        raise ValueError(f"unsupported shape {tuple(x.shape)}: no empty dimension, D even and up to 256")
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be 'interleaved' or 'halves', got {layout!r}")
    axes, total = len(axis_pairs), sum(axis_pairs)
    if not 1 <= axes <= 4 or min(axis_pairs) < 0 or total > D // 2:
        raise ValueError(f"axis_pairs {list(axis_pairs)} must be 1 to 4 counts of at most {D // 2} pairs in all")
    device, kind = x.device, _POSITIONS.get(positions.dtype)
    if kind is None:
        raise ValueError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    if positions.shape == (L, axes):
        apart = 0
    elif positions.shape == (B, L, axes):
        apart = L * axes
    else:
        raise ValueError(f"positions must be [L, axes] or [B, L, axes], got {tuple(positions.shape)}")
    if positions.device != device:
        raise ValueError(f"positions must be on {device}")
    inv_freq = _check(inv_freq, "inv_freq", (total,), torch.float32, device).contiguous()
    gamma = _param(gamma, "gamma", (H, D), device)
    how = (code, kind, apart, B, L, H, D, _I32[axes].pack(*axis_pairs), axes, _LAYOUTS[layout])
    return positions.contiguous(), inv_freq, gamma, how


_I32 = [struct.Struct(f"{n}i") for n in range(5)]


def _out_like(out, x, name):
    """An output of x's shape and type, and its strides: `out` if given (unit last stride), a new one
    otherwise."""
    if out is None:
        out = x.new_empty(x.shape)
        return out, out.stride()
    _check(out, name, x.shape, x.dtype, x.device)
    st = out.stride()
    if st[-1] != 1 and out.shape[-1] != 1:
        raise ValueError(f"{name} needs a contiguous last dimension")
    if any(n > 1 and s == 0 for n, s in zip(out.shape, st)):
        raise ValueError(f"{name} must not be expanded")
    return out, st


def axis_rope(x, positions, inv_freq, *, axis_pairs, gamma=None, layout="interleaved", out=None):
    """Rotates x [B, L, H, D] by its tokens' positions [L, axes] (or [B, L, axes]).

    The first sum(axis_pairs) pairs of each head turn, axis_pairs[a] of them by axis a's
    position times their entry of ``inv_freq``; a pair is elements (2p, 2p+1) ("interleaved")
    or (p, P+p) ("halves").  With ``gamma`` [H, D] the rotated vector r becomes
    r * sqrt(D) / max(|r|, 1e-12) * gamma.  ``out`` may be x itself."""
    positions, inv_freq, gamma, how = _rope_args(x, positions, inv_freq, axis_pairs, gamma, layout)
    x, xs = _rows(x)
    y, ys = _out_like(out, x, "out")
    lib = _lib(x.device)
    _ok(lib, lib.triposplat_b200_axis_rope(
        x.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), _ptr(gamma), y.data_ptr(),
        _I64[6].pack(*xs[:3], *ys[:3]), *how), "axis_rope")
    return y


def axis_rope_backward(dy, x, positions, inv_freq, *, axis_pairs, gamma=None, layout="interleaved",
                       out=None):
    """Gradients (dx, dgamma) of ``axis_rope`` at x (read only with ``gamma``; dgamma is None
    without).  ``out`` receives dx and may be dy itself."""
    positions, inv_freq, gamma, how = _rope_args(dy, positions, inv_freq, axis_pairs, gamma, layout)
    dy, ds = _rows(dy)
    dx, gs = _out_like(out, dy, "out")
    px, xs, dgamma = None, (0, 0, 0), None
    if gamma is not None:
        x, xs = _rows(_check(x, "x", dy.shape, dy.dtype, dy.device))
        px, dgamma = x.data_ptr(), torch.empty_like(gamma)
    lib = _lib(dy.device)
    _ok(lib, lib.triposplat_b200_axis_rope_backward(
        dy.data_ptr(), px, positions.data_ptr(), inv_freq.data_ptr(), _ptr(gamma), dx.data_ptr(), _ptr(dgamma),
        _I64[9].pack(*ds[:3], *xs[:3], *gs[:3]), *how), "axis_rope_backward")
    return dx, dgamma


# ------------------------------------------------------------- norms with gate and residual
def _norm_args(x, y, gate, scale, shift, pre, pre_weight, post, post_weight):
    if x.dim() != 3 or x.dtype not in _DTYPES:
        raise ValueError("x must be [B, L, C] in float32, bfloat16 or float16")
    B, L, C = x.shape
    if not (B and L and C) or C > 8192 or B > 65535:
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
    (x, xs), (y, ys) = _rows(x), _rows(y)
    B, L, C = x.shape
    z = x.new_empty((B, L, C))
    h = x.new_empty((B, L, C)) if pre is not None else None
    stats = torch.empty((B, L, 4), dtype=torch.float32, device=x.device)
    lib = _lib(x.device)
    _ok(lib, lib.triposplat_b200_norm_gate(
        x.data_ptr(), y.data_ptr(), _I64[4].pack(*xs[:2], *ys[:2]), _ptr(gate), _ptr(scale), _ptr(shift),
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
    zs = hs = (0, 0)
    if dz is not None:
        dz, zs = _rows(_check(dz, "dz", x.shape, x.dtype, x.device))
    if dh is not None:
        dh, hs = _rows(_check(dh, "dh", x.shape, x.dtype, x.device))
    (x, xs), (y, ys) = _rows(x), _rows(y)
    B, L, C = x.shape
    stats = _check(stats, "stats", (B, L, 4), torch.float32, x.device).contiguous()
    g = {"x": x.new_empty((B, L, C)), "y": x.new_empty((B, L, C))}
    for name, t in (("gate", gate), ("scale", scale), ("shift", shift), ("pre_weight", wpre),
                    ("post_weight", wpost)):
        g[name] = None if t is None else torch.empty_like(t)
    lib = _lib(x.device)
    _ok(lib, lib.triposplat_b200_norm_gate_backward(
        _ptr(dz), _ptr(dh), x.data_ptr(), y.data_ptr(), _I64[8].pack(*xs[:2], *ys[:2], *zs[:2], *hs[:2]),
        stats.data_ptr(), _ptr(gate), _ptr(scale),
        _ptr(wpre), _ptr(wpost), g["x"].data_ptr(), g["y"].data_ptr(), _ptr(g["gate"]), _ptr(g["scale"]),
        _ptr(g["shift"]), _ptr(g["pre_weight"]), _ptr(g["post_weight"]), _DTYPES[x.dtype], B, L, C, _KINDS[pre],
        _KINDS[post], float(residual_scale)), "norm_gate_backward")
    return g


# --------------------------------------------------------------------------------- attention
def _attention_args(q, k, v, key_bias):
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q, k, v must be [B, H, L, 64]")
    B, H, Lq, D = q.shape
    Lk, dev = k.shape[2], q.device
    if D != 64 or not (B and H and Lq and Lk):
        raise ValueError(f"unsupported shapes {tuple(q.shape)}, {tuple(k.shape)}: head_dim 64, no empty dimension")
    _check(q, "q", q.shape, torch.float32, dev)
    _check(k, "k", (B, H, Lk, 64), torch.float32, dev)
    _check(v, "v", k.shape, torch.float32, dev)
    if key_bias is None:
        return None, 1, 1, B, H, Lq, Lk
    shape = key_bias.shape
    if shape not in ((Lk,), (B, Lk), (B, H, Lk)):
        raise ValueError(f"key_bias must be [Lk], [B, Lk] or [B, H, Lk], got {tuple(shape)}")
    return (_param(key_bias, "key_bias", shape, dev), B if len(shape) > 1 else 1, H if len(shape) > 2 else 1,
            B, H, Lq, Lk)


def _token_major(like, B, H, L):
    """A new [B, H, L, 64] in token-major storage [B, L, H, 64]."""
    return like.new_empty_strided((B, H, L, 64), (L * H * 64, 64, H * 64, 1))


def attention_forward(q, k, v, *, key_bias=None):
    """softmax(q k^T / 8 + key_bias) v on q [B, H, Lq, 64] and k, v [B, H, Lk, 64] (float32), key_bias
    [Lk], [B, Lk] or [B, H, Lk].  A key with a bias of -inf does not exist; a query without keys
    gives zeros.  Returns (out, stats): out [B, H, Lq, 64] in token-major storage
    ([B, Lq, H, 64], what the out-projection reads), stats [B, H, Lq + 1, 2] for the backward pass.
    Heads shared by several queries' heads are passed expanded."""
    key_bias, bias_b, bias_h, B, H, Lq, Lk = _attention_args(q, k, v, key_bias)
    (q, qs), (k, ks), (v, vs) = _rows(q), _rows(k), _rows(v)
    out = _token_major(q, B, H, Lq)
    stats = q.new_empty((B, H, Lq + 1, 2))
    lib = _lib(q.device)
    _ok(lib, lib.triposplat_b200_attention_forward(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _I64[9].pack(*qs[:3], *ks[:3], *vs[:3]), _ptr(key_bias), bias_b,
        bias_h, out.data_ptr(), stats.data_ptr(), B, H, Lq, Lk), "attention_forward")
    return out, stats


def attention_backward(dout, q, k, v, out, stats, *, key_bias=None, grads=None, bias_grad=True):
    """Gradients (dq, dk, dv, dbias) of ``attention_forward`` with the incoming dout [B, H, Lq, 64].

    ``grads`` may name the three tensors to write (e.g. slices of a packed gradient); otherwise they
    are new, in token-major storage.  dbias has key_bias's shape (None without a bias or with
    ``bias_grad=False``)."""
    key_bias, bias_b, bias_h, B, H, Lq, Lk = _attention_args(q, k, v, key_bias)
    dev = q.device
    dout, gs = _rows(_check(dout, "dout", q.shape, torch.float32, dev))
    out, os = _rows(_check(out, "out", q.shape, torch.float32, dev))
    stats = _check(stats, "stats", (B, H, Lq + 1, 2), torch.float32, dev).contiguous()
    (q, qs), (k, ks), (v, vs) = _rows(q), _rows(k), _rows(v)
    if grads is None:
        dq, dk, dv = _token_major(q, B, H, Lq), _token_major(k, B, H, Lk), _token_major(v, B, H, Lk)
        dqs, dks, dvs = dq.stride(), dk.stride(), dv.stride()
    else:
        (dq, dqs), (dk, dks), (dv, dvs) = (_out_like(g, like, "grads") for g, like in zip(grads, (q, k, v), strict=True))
    dbias = torch.empty_like(key_bias) if key_bias is not None and bias_grad else None
    strides = _I64[24].pack(*gs[:3], *qs[:3], *ks[:3], *vs[:3], *os[:3], *dqs[:3], *dks[:3], *dvs[:3])
    lib = _lib(dev)
    _ok(lib, lib.triposplat_b200_attention_backward(
        dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), stats.data_ptr(), strides,
        _ptr(key_bias), bias_b, bias_h, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dbias), B, H, Lq, Lk),
        "attention_backward")
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
