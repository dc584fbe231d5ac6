"""attention without a GPU: the C ABI refuses bad arguments before any device work, the workspace queries, and what the Python
entry points refuse"""
import ctypes

import pytest
import torch

import spanqr_amd as sp
from spanqr_amd import _lib

EINVAL = -1
PTR = ctypes.c_void_p(4096)   # never read: every call here is refused first


def strides(batch=64 * 4 * 10, row=64 * 4, head=64):
    return (ctypes.c_long * 3)(batch, row, head)


BAD_SHAPES = [dict(type=0), dict(type=3), dict(B=-1), dict(Hk=0), dict(G=0), dict(D=0), dict(D=4), dict(D=136), dict(D=60), dict(Tq=-1),
              dict(Tk=-1), dict(Tk=1 << 30), dict(Tq=1 << 29), dict(G=1 << 31), dict(B=1 << 40), dict(B=1 << 23), dict(Tq=1 << 28, Hk=8),
              dict(qs=PTR), dict(ks=PTR), dict(qs=PTR, ks=PTR, lens=PTR), dict(window=-1, causal=1), dict(window=3, causal=0), dict(scale=0.0), dict(scale=-1.0),
              dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(q=None), dict(k=None), dict(v=None), dict(q=ctypes.c_void_p(4098)),
              dict(q_str=strides(row=65)), dict(q_str=strides(head=1 << 24)), dict(k_str=strides(row=-8)), dict(v_str=strides(batch=4)),
              dict(k_str=None)]


def test_forward_refusals():
    def call(type=1, B=2, Hk=2, G=2, D=64, Tq=10, Tk=10, q=PTR, k=PTR, v=PTR, q_str=strides(), k_str=strides(), v_str=strides(), qs=None,
             ks=None, lens=None, max_q=0, max_k=0, causal=1, window=0, scale=1.0, out=PTR, ws=None, nbytes=0):
        return _lib.lib().spanqr_attention(type, B, Hk, G, D, Tq, Tk, q, q_str, k, k_str, v, v_str, qs, ks, lens, max_q, max_k, causal,
                                           window, scale, out, None, ws, nbytes, None)

    for kw in [*BAD_SHAPES, dict(out=None), dict(out=ctypes.c_void_p(8)), dict(Tk=4096), dict(Tk=4096, ws=PTR, nbytes=100)]:
        assert call(**kw) == EINVAL, kw
        assert b"attention" in _lib.lib().spanqr_last_error()
    assert call(Tq=0, q=None, out=None) == 0 and call(B=0, q=None, out=None) == 0


def test_backward_refusals():
    need = _lib.lib().spanqr_attention_backward_workspace(2, 2, 2, 64, 10, 10, 0, 0, 0)
    assert need == 8 * 2 * 10 * 4 + 4 * 2 * 2 * (1 + 1)

    def call(type=1, B=2, Hk=2, G=2, D=64, Tq=10, Tk=10, do=PTR, q=PTR, k=PTR, v=PTR, o=PTR, do_str=strides(), q_str=strides(),
             k_str=strides(), v_str=strides(), o_str=strides(), lse=PTR, qs=None, ks=None, lens=None, causal=1, window=0, scale=1.0, dq=PTR, dk=PTR,
             dv=PTR, ws=PTR, nbytes=need):
        return _lib.lib().spanqr_attention_backward(type, B, Hk, G, D, Tq, Tk, do, do_str, q, q_str, k, k_str, v, v_str, o, o_str, lse,
                                                    qs, ks, lens, 0, 0, causal, window, scale, dq, dk, dv, ws, nbytes, None)

    for kw in [*BAD_SHAPES, dict(do=None), dict(o=None), dict(do_str=strides(row=4)), dict(o_str=strides(head=12)), dict(lse=None),
               dict(ws=None), dict(nbytes=need - 1), dict(dk=None), dict(dv=None), dict(dq=ctypes.c_void_p(8)),
               dict(dk=ctypes.c_void_p(24)), dict(type=2, Tq=0, ws=None), dict(Tq=0, nbytes=4 * 2 * 2 * 2 - 1)]:
        assert call(**kw) == EINVAL, kw
        assert b"attention_backward" in _lib.lib().spanqr_last_error()
    assert call(B=0, ws=None, nbytes=0, lse=None) == 0


def test_workspace():
    f = _lib.lib().spanqr_attention_workspace
    assert f(16, 12, 1, 64, 1024, 1024, 0, 0, 0) == 0            # enough workgroups
    assert f(1, 8, 5, 128, 1, 8191, 0, 0, 0) == 4 * 63 * 40 * 130   # 63 pieces of 128 keys at least
    assert f(1, 1, 1, 64, 1, 100, 0, 0, 0) == 0                  # too few keys to split
    assert f(0, 8, 5, 128, 1, 8191, 0, 0, 0) == 0
    assert f(1, 8, 5, 129, 1, 8191, 0, 0, 0) == EINVAL
    # packed: by the longest sequence, where it is known
    assert f(32, 2, 8, 128, 32, 70000, 1, 1, 4096) == 4 * 8 * 32 * 16 * 130
    assert f(4, 1, 1, 64, 4, 400, 1, 1, 100) == 0
    # hints far below what there is do not multiply what is held for all rows
    assert f(1, 2, 1, 64, 1 << 20, 1 << 20, 1, 1, 1 << 20) == 0
    g = _lib.lib().spanqr_attention_backward_workspace
    assert g(1, 1, 1, 64, 1 << 20, 1 << 20, 1, 1, 1) == 8 * (1 << 20) + 4 * 2
    # few tiles: 11 of dQ's rows in 5 parts (22 tiles of keys, four each at least), 22 of dK's and dV's in 5 (22 of rows)
    assert g(1, 1, 8, 64, 171, 1362, 0, 0, 0) == (8 * 1368 + 4 * (11 + 11) + 15) // 16 * 16 + 4 * 64 * (5 * 1368 + 2 * 5 * 1362)
    assert g(0, 1, 8, 64, 171, 1362, 1, 0, 0) == 8 * 1368 and f(0, 1, 8, 64, 171, 1362, 1, 0, 0) == 0


def test_python_refusals_on_the_host():
    q = torch.zeros(1, 4, 2, 16, dtype=torch.bfloat16)
    for f in (lambda: sp.attention(q, q, q), lambda: sp.attention_backward(q, q, q, q, q, q[..., 0].float())):
        with pytest.raises(TypeError, match="GPU"):
            f()


def test_packed_calls_without_hints():
    """many sequences whose longest one nobody names: what is launched goes by the rows there are"""
    f, g = _lib.lib().spanqr_attention_workspace, _lib.lib().spanqr_attention_backward_workspace
    for B, Hk, G, T in ((512, 8, 1, 1 << 19), (1000, 8, 1, 1 << 20), (1024, 8, 1, 1 << 18), (256, 8, 5, 1 << 17), (1 << 15, 4, 2, 1 << 20)):
        assert f(B, Hk, G, 128, T, T, 1, 0, 0) == 0, (B, Hk, G, T)
        # two numbers a row, and a maximum for each slot of the list
        assert g(B, Hk, G, 128, T, T, 1, 0, 0) == 8 * T * Hk * G + 4 * Hk * (T * G // 128 + B + T // 128 + B), (B, Hk, G, T)
    assert f(1 << 24, 1, 1, 128, 1 << 24, 1 << 24, 1, 0, 0) == EINVAL   # a workgroup for each is too many
    assert b"too many workgroups" in _lib.lib().spanqr_last_error()
    # more tiles than a launch takes workgroups: each goes over several
    assert f((1 << 23) - 1, 1, 129, 8, 1, 4, 0, 0, 0) == 0


def test_parts_by_what_runs_at_once():
    """640 tiles of dQ, 64 wide: fewer than the 768 that run at once in bf16, more than fp16's 512"""
    L = _lib.lib()
    shape = 5, 8, 1, 64, 2048, 2048
    stat = 8 * 5 * 2048 * 8 + 4 * 5 * 8 * (16 + 16)
    row = 4 * 5 * 2048 * 8 * 64   # bytes of a part
    for type, parts in ((1, 2), (2, 0)):   # (dK and dV have 1280 tiles of 64 keys)
        assert L.spanqr_attention_backward(type, *shape, PTR, strides(), PTR, strides(), PTR, strides(), PTR, strides(), PTR, strides(), PTR,
                                           None, None, None, 0, 0, 1, 0, 1.0, PTR, PTR, PTR, None, 0, None) == EINVAL
        need = int(L.spanqr_last_error().split(b"needs ")[1].split()[0])
        assert need == stat + parts * row
        assert need <= L.spanqr_attention_backward_workspace(*shape, 0, 0, 0)
