"""Norms with gate and residual at widths that are no multiple of four: contiguous tensors (rows start between
access boundaries), padded rows of the same remainder, and rows of different ones; the memory around the rows holds
NaN.  Against the definition in 64 bits.

Tolerance, 2-norms over a result.  An element is at most some 64 roundings (u = 2^-24) of its row's level from its
definition, and half a unit of its own type: U + 64 u = U + 2^-18 of the result's norm.  A column sum of n terms of
random sign has n additions of at most the sum of magnitudes, sqrt(n) times the level of the sum:
(64 + n) sqrt(n) u.
"""
import math

import pytest
import torch

from test_train_ops_gpu import TYPES, U32, UNIT, norm_ref, randn

pytestmark = pytest.mark.gpu

WIDTHS = [5, 7, 93, 125, 126, 127, 129, 255, 509, 510, 511, 513, 1111, 2047, 2050, 4093, 4094, 4095, 8189, 8190, 8191]


def placed(t, layout):
    """A copy of t [B, L, C] in a buffer of NaN: "tight" rows on a 16-byte boundary, "padded" rows 4 (mod 16)
    elements apart from tight, "odd" rows one element apart, off the boundary, or "tail", tight up to the
    buffer's end."""
    B, L, C = t.shape
    step = {"tight": C, "tail": C, "padded": C + 20, "odd": C + 1}[layout]
    buf = torch.full((B * L * step + 128,), math.nan, dtype=t.dtype, device=t.device)
    at = 65 if layout == "odd" else 64
    if layout == "tail":
        buf = buf[:64 + B * L * C]
    v = buf.as_strided((B, L, C), (L * step, step, 1), at)
    v.copy_(t)
    return v


def close(got, ref, name, unit, n=0):
    assert torch.isfinite(got).all(), name
    bound = ((64 + n) * math.sqrt(n) * U32 if n else unit + 64 * U32) * ref.norm().item()
    err = (got.double() - ref).norm().item()
    assert err <= bound, f"{name}: {err:.3e} > {bound:.3e}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["tight", "padded", "odd", "tail"])
@pytest.mark.parametrize("C", WIDTHS)
def test_widths(C, layout, dtype):
    import train_ops

    B, L = (2, 9) if C % 2 else (3, 6)
    x, y, dz, dh = (placed(randn(s, B, L, C, dtype=dtype), layout) for s in range(1, 5))
    p = dict(gate=randn(5, B, C), scale=randn(6, B, C, scale=0.3), shift=randn(7, B, C),
             pre_weight=1 + randn(8, C, scale=0.1), post_weight=1 + randn(9, C, scale=0.1))
    kinds = dict(pre="layer" if C % 3 else "rms", post="rms" if C % 3 else "layer")
    z, h, stats = train_ops.norm_gate(x, y, **p, **kinds, residual_scale=0.7, eps=1e-5)
    got = train_ops.norm_gate_backward(dz, dh, x, y, stats, **p, **kinds, residual_scale=0.7, eps=1e-5)
    leaf = {k: v.double().requires_grad_() for k, v in dict(p, x=x, y=y).items()}
    rz, rh = norm_ref(leaf["x"], leaf["y"], leaf, kinds["pre"], kinds["post"], 0.7, 1e-5)
    ref = dict(zip(leaf, torch.autograd.grad((rz * dz.double()).sum() + (rh * dh.double()).sum(), list(leaf.values()))))
    close(z, rz.detach(), "z", UNIT[dtype])
    close(h, rh.detach(), "h", UNIT[dtype])
    for k in ("x", "y"):
        close(got[k], ref[k], k, UNIT[dtype])
    for k in p:
        close(got[k], ref[k], k, UNIT[dtype], n=L if p[k].dim() == 2 else B * L)


@pytest.mark.parametrize("L", [1, 3, 4, 5, 700, 4001])
def test_many_rows(L):
    """Row groups of several rows, the groups' number not a divisor of theirs; the same bits again."""
    import train_ops

    B, C = 2, 333
    x, y, dz, dh = (randn(s, B, L, C) for s in range(1, 5))
    how = dict(gate=randn(5, B, C), pre="rms", post="layer")
    z, h, stats = train_ops.norm_gate(x, y, **how)
    rz, rh = norm_ref(x.double(), y.double(), {"gate": how["gate"].double()}, "rms", "layer", 1.0, 1e-6)
    close(z, rz, "z", U32)
    close(h, rh, "h", U32)
    first, again = (train_ops.norm_gate_backward(dz, dh, x, y, stats, **how) for _ in range(2))
    assert all(torch.equal(first[k], again[k]) for k in ("x", "y", "gate"))
    leaf = {k: v.double().requires_grad_() for k, v in dict(x=x, y=y, gate=how["gate"]).items()}
    rz, rh = norm_ref(leaf["x"], leaf["y"], leaf, "rms", "layer", 1.0, 1e-6)
    ref = dict(zip(leaf, torch.autograd.grad((rz * dz.double()).sum() + (rh * dh.double()).sum(), list(leaf.values()))))
    close(first["x"], ref["x"], "x", U32)
    close(first["y"], ref["y"], "y", U32)
    close(first["gate"], ref["gate"], "gate", U32, n=L)
