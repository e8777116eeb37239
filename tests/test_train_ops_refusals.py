"""Status codes of the training operators' C entries for arguments they refuse before they look
at a device."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    import _native
    import build_lib

    build_lib.build()
    return _native.load()


P = 4096  # stands for a device pointer that is never reached


def strides(n):
    return (ctypes.c_int64 * n)(*([64] * n))


def rope(lib, x=P, dtype=0, pos_type=0, B=1, L=1, H=1, D=64, pairs=(32,), layout=0):
    return lib.triposplat_b200_axis_rope(x, P, P, None, P, strides(6), dtype, pos_type, 0, B, L, H, D,
                                         (ctypes.c_int * len(pairs))(*pairs), len(pairs), layout)


def test_rope(lib):
    assert rope(lib, x=None) == -1
    for bad in (dict(B=0), dict(L=0), dict(H=0), dict(D=0), dict(D=63), dict(D=258), dict(pairs=(1,) * 5), dict(B=65536)):
        assert rope(lib, **bad) == -2, bad
    for bad in (dict(dtype=3), dict(dtype=-1), dict(pos_type=3), dict(pairs=(20, 13)), dict(pairs=(-1,)), dict(layout=2)):
        assert rope(lib, **bad) == -3, bad
    assert rope(lib, x=P + 2) == -4 and rope(lib, x=P + 1, dtype=1) == -4


def norm(lib, x=P, scale=None, shift=None, wpre=None, h=P, stats=P, dtype=0, B=1, L=1, C=8, pre=1, post=0):
    return lib.triposplat_b200_norm_gate(x, P, strides(4), None, scale, shift, wpre, None, P, h, stats, dtype, B, L, C,
                                         pre, post, 1.0, 1e-6)


def test_norm(lib):
    for bad in (dict(x=None), dict(h=None), dict(stats=None), dict(scale=P)):
        assert norm(lib, **bad) == -1, bad
    for bad in (dict(B=0), dict(L=0), dict(C=0), dict(C=8193), dict(B=65536)):
        assert norm(lib, **bad) == -2, bad
    for bad in (dict(dtype=3), dict(pre=3), dict(post=-1), dict(pre=0, wpre=P), dict(pre=0, scale=P, shift=P)):
        assert norm(lib, **bad) == -3, bad
    assert norm(lib, stats=P + 4) == -4 and norm(lib, x=P + 2) == -4


def test_clip(lib):
    def call(ptr=P, size=4, dtype=0, count=1, most=1.0, norm=P):
        return lib.triposplat_b200_clip_grad_norm((ctypes.c_void_p * 1)(ptr), None, (ctypes.c_int64 * 1)(size),
                                                  (ctypes.c_int * 1)(dtype), count, most, norm)

    assert call(ptr=None) == -1 and call(norm=None) == -1
    assert call(count=-1) == -2 and call(most=-1.0) == -2 and call(most=float("nan")) == -2 and call(size=-1) == -2
    assert call(dtype=3) == -3 and call(ptr=P + 2) == -4


def test_attention(lib):
    def fwd(q=P, bias=None, bb=1, bh=1, out=P, stats=P, B=2, H=2, Lq=1, Lk=1):
        return lib.triposplat_b200_attention_forward(q, P, P, strides(9), bias, bb, bh, out, stats, B, H, Lq, Lk)

    def bwd(dq=P, dbias=None, bias=None, B=2, Lq=1, Lk=1, dout=P):
        return lib.triposplat_b200_attention_backward(dout, P, P, P, P, P, strides(24), bias, 1, 1, dq, P, P, dbias, B, 2,
                                                      Lq, Lk)

    assert fwd(q=None) == -1 and fwd(stats=None) == -1 and bwd(dq=None) == -1 and bwd(dbias=P) == -1
    for bad in (dict(B=0), dict(H=0), dict(Lq=0), dict(Lk=0), dict(B=40000), dict(Lq=64 * 65535 + 1)):
        assert fwd(**bad) == -2, bad
    assert bwd(B=0) == -2 and bwd(Lk=0) == -2 and bwd(Lq=4000000, Lk=4000000) == -2
    assert fwd(bias=P, bb=3) == -3 and fwd(bias=P, bh=3) == -3
    assert fwd(q=P + 2) == -4 and fwd(out=P + 4) == -4 and fwd(stats=P + 4) == -4 and bwd(dout=P + 1) == -4
