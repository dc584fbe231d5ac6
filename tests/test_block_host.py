"""block_norm and dropout without a GPU: the C ABI refuses bad arguments before any device work, and the Python entry points
refuse what they do not take"""
import ctypes

import pytest
import torch

import spanqr_amd as sp
from spanqr_amd import _lib

EINVAL = -1
PTR = ctypes.c_void_p(4096)   # never read: every call here is refused first


def test_dropout_refusals():
    def call(type=1, rows=2, D=8, x=PTR, ldx=8, p=0.5, y=PTR):
        return _lib.lib().spanqr_dropout(type, rows, D, x, ldx, p, 1, None, 0, y, None)

    for kw in [dict(type=3), dict(rows=-1), dict(D=0), dict(D=(1 << 32) + 1), dict(rows=1 << 40), dict(x=None), dict(y=None),
               dict(ldx=7), dict(p=1.0), dict(p=-0.1), dict(p=float("nan")), dict(p=1 - 2.0 ** -17)]:
        assert call(**kw) == EINVAL, kw
        assert b"dropout" in _lib.lib().spanqr_last_error()
    assert call(rows=0, x=None, y=None) == 0


def test_block_norm_refusals():
    def call(type=1, wtype=1, act=2, rows=2, D=8, x=PTR, ldx=8, r=PTR, ldr=8, g=None, ldg=0, p=0.0, h=PTR, y=PTR):
        return _lib.lib().spanqr_block_norm(type, wtype, act, rows, D, x, ldx, r, ldr, g, ldg, None, None, 1e-6, 1.0, None, p, 0,
                                            None, 0, h, y, None)

    for kw in [dict(type=-1), dict(wtype=3), dict(act=3), dict(act=-1), dict(rows=-1), dict(D=0), dict(D=(1 << 24) + 1),
               dict(x=None), dict(r=None), dict(h=None), dict(y=None), dict(ldx=7), dict(ldr=7), dict(g=PTR, ldg=7), dict(p=1.0)]:
        assert call(**kw) == EINVAL, kw
        assert b"block_norm" in _lib.lib().spanqr_last_error()
    assert call(rows=0, x=None, r=None, h=None, y=None) == 0


def test_block_norm_backward_refusals():
    f = _lib.lib().spanqr_block_norm_backward_workspace
    need = f(4, 64)
    assert need == 4 * 129 * 1   # four rows of up to 128 elements are one workgroup's
    assert f(-1, 64) == f(4, 0) == f(4, (1 << 24) + 1) == EINVAL
    assert f(1 << 20, 2048) <= 4 * 1024 * 4097

    def call(type=0, wtype=0, act=0, rows=4, D=64, dy=PTR, lddy=64, dh=PTR, lddh=64, x=PTR, ldx=64, h=PTR, ldh=64, g=None,
             ldg=64, p=0.0, dx=PTR, dr=PTR, dg=None, dw=PTR, ws=PTR, nbytes=need):
        return _lib.lib().spanqr_block_norm_backward(type, wtype, act, rows, D, dy, lddy, dh, lddh, x, ldx, h, ldh, g, ldg, None,
                                                     PTR, 1e-6, 1.0, None, p, 0, None, 0, dx, dr, dg, None, dw, None, ws, nbytes,
                                                     None)

    for kw in [dict(type=5), dict(wtype=-1), dict(act=7), dict(rows=-1), dict(D=0), dict(x=None), dict(h=None), dict(dx=None),
               dict(dr=None), dict(g=PTR), dict(dg=PTR), dict(ws=None), dict(nbytes=need - 1), dict(lddy=63), dict(lddh=63),
               dict(ldx=63), dict(ldh=63), dict(g=PTR, dg=PTR, ldg=63), dict(p=-1.0)]:
        assert call(**kw) == EINVAL, kw
        assert b"block_norm_backward" in _lib.lib().spanqr_last_error()


def test_python_refusals_on_the_host():
    x = torch.zeros(4, 8)
    for f in (lambda: sp.dropout(x, 0.5, 1), lambda: sp.block_norm(x, x), lambda: sp.block_norm_backward(x, x, x, x)):
        with pytest.raises(TypeError, match="GPU"):
            f()
    with pytest.raises(ValueError):
        sp.dropout(1.0, 0.5, 1)
