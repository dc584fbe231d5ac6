"""The training operators without a GPU: the C ABI refuses bad arguments before any device work, its workspace queries
keep their bounds, and the Python entry points refuse what they do not take."""
import ctypes

import pytest
import torch

import spanqr_amd as sp
from spanqr_amd import _lib

EINVAL = -1
PTR = ctypes.c_void_p(4096)   # never read: every call here is refused first


def lib():
    return _lib.lib()


def test_rms_norm_refusals():
    f = lib().spanqr_rms_norm

    def call(type=1, wtype=1, quant=0, rows=2, D=8, x=PTR, ldx=8, r=None, ldr=0, w=None, h=None, y=PTR, scale=None):
        return f(type, wtype, quant, rows, D, x, ldx, r, ldr, w, 1e-6, h, y, scale, None)

    bad = [dict(type=7), dict(wtype=-1), dict(quant=3), dict(rows=-1), dict(D=0), dict(D=(1 << 24) + 1), dict(x=None),
           dict(y=None), dict(r=PTR, ldr=8), dict(h=PTR), dict(quant=1), dict(scale=PTR), dict(ldx=7),
           dict(r=PTR, h=PTR, ldr=7), dict(rows=1 << 40, D=1 << 20)]
    for kw in bad:
        assert call(**kw) == EINVAL, kw
        assert b"rms_norm" in lib().spanqr_last_error()
    assert call(rows=0, x=None, y=None) == 0   # nothing to do, nothing read


def test_rms_norm_backward_refusals():
    f = lib().spanqr_rms_norm_backward
    need = lib().spanqr_rms_norm_backward_workspace(4, 64)
    assert need >= 4 * 64

    def call(type=0, wtype=0, rows=4, D=64, dy=PTR, lddy=64, h=PTR, ldh=64, w=PTR, dh=None, lddh=0, dx=PTR, dw=PTR,
             ws=PTR, nbytes=need):
        return f(type, wtype, rows, D, dy, lddy, h, ldh, w, dh, lddh, 1e-6, dx, dw, ws, nbytes, None)

    for kw in [dict(type=3), dict(rows=-2), dict(D=0), dict(dy=None), dict(h=None), dict(dx=None), dict(ws=None),
               dict(nbytes=need - 1), dict(lddy=63), dict(ldh=1), dict(dh=PTR, lddh=63)]:
        assert call(**kw) == EINVAL, kw
    assert lib().spanqr_rms_norm_backward_workspace(-1, 64) == EINVAL
    assert lib().spanqr_rms_norm_backward_workspace(4, 0) == EINVAL
    # bounded in the rows
    assert lib().spanqr_rms_norm_backward_workspace(1 << 30, 64) <= 4 * 64 * 4096


def test_clip_refusals():
    n = 2
    ptrs = (ctypes.c_void_p * n)(4096, 8192)
    numel = (ctypes.c_long * n)(5, 0)
    types = (ctypes.c_int * n)(0, 1)
    need = lib().spanqr_grad_norm_workspace(n)
    assert need > 0 and lib().spanqr_grad_norm_workspace(-1) == EINVAL
    g = lib().spanqr_grad_norm
    c = lib().spanqr_clip_grad_norm
    assert g(-1, ptrs, numel, types, PTR, PTR, need, None) == EINVAL
    assert g(n, None, numel, types, PTR, PTR, need, None) == EINVAL
    assert g(n, ptrs, numel, types, None, PTR, need, None) == EINVAL
    assert g(n, ptrs, numel, types, PTR, None, need, None) == EINVAL
    assert g(n, ptrs, numel, types, PTR, PTR, need - 1, None) == EINVAL
    assert g(n, ptrs, (ctypes.c_long * n)(5, -1), types, PTR, PTR, need, None) == EINVAL
    assert g(n, ptrs, numel, (ctypes.c_int * n)(0, 9), PTR, PTR, need, None) == EINVAL
    assert g(n, (ctypes.c_void_p * n)(None, 4096), numel, types, PTR, PTR, need, None) == EINVAL
    assert c(n, ptrs, numel, types, None, types, 1.0, PTR, PTR, need, None) == EINVAL
    assert c(n, ptrs, numel, types, ptrs, None, 1.0, PTR, PTR, need, None) == EINVAL
    for bad in (-1.0, float("nan")):
        assert c(n, ptrs, numel, types, ptrs, types, bad, PTR, PTR, need, None) == EINVAL
        assert b"max_norm" in lib().spanqr_last_error()


def test_loss_refusals():
    need = lib().spanqr_linear_cross_entropy_workspace(1, 4, 64, 100, 3, 1 << 30)
    assert need > 0

    def call(type=1, red=2, N=4, H=64, V=100, x=PTR, ldx=64, w=PTR, ldw=64, t=PTR, loss=PTR, dx=PTR, dw=PTR, ws=PTR,
             nbytes=need):
        return lib().spanqr_linear_cross_entropy(type, red, N, H, V, x, ldx, w, ldw, t, -100, None, None, loss, None, dx,
                                                 dw, ws, nbytes, None)

    for kw in [dict(type=0), dict(type=5), dict(red=3), dict(N=-1), dict(H=0), dict(V=0), dict(x=None), dict(w=None),
               dict(t=None), dict(loss=None), dict(ws=None), dict(ldx=63), dict(ldw=63), dict(nbytes=need - 256),
               dict(V=(1 << 24) + 1)]:
        assert call(**kw) == EINVAL, kw
        assert b"linear_cross_entropy" in lib().spanqr_last_error()


@pytest.mark.parametrize("grads", [0, 1, 2, 3])
def test_loss_workspace_is_bounded(grads):
    """what the query gives stays within most_bytes once that holds 256 tokens and the sums of dW, and does not grow
    with the tokens"""
    f = lib().spanqr_linear_cross_entropy_workspace
    H, V, most = 1024, 50257, 600 << 20
    sizes = [f(1, N, H, V, grads, most) for N in (1, 256, 1000, 8192, 100000, 1 << 20)]
    assert all(0 < s <= most for s in sizes), sizes
    assert f(1, 256, H, V, grads, 0) == f(1, 256, H, V, grads, most)


def test_python_refusals_on_the_host():
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    w = torch.zeros(16, 8, dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64)
    for f in (lambda: sp.linear_cross_entropy(x, w, t), lambda: sp.linear_cross_entropy_grad(x, w, t),
              lambda: sp.rms_norm(x), lambda: sp.rms_norm_backward(x, x), lambda: sp.grad_norm([x]),
              lambda: sp.clip_grad_norm([x], 1.0), lambda: sp.rms_norm(x.double())):
        with pytest.raises(TypeError):
            f()
    for f in (lambda: sp.rms_norm([1.0]), lambda: sp.grad_norm([None])):
        with pytest.raises(ValueError):
            f()
