"""What stands between two blocks of a model: the norms behind one and in front of the next, fused with the gate, dropout and
the scaled addition to the residual stream, and dropout alone, through the native library (csrc/block.hip). No counterpart
in the reference; the blocks' weights are what the optimizer that calls orth works on.
"""
from collections import namedtuple

import torch

from . import _lib
from .tensors import TYPES, check_like, check_same, check_tensor, like, no_tangents, on, once, rows_of, workspace

GATES = {None: _lib.GATE_LINEAR, "sigmoid": _lib.GATE_SIGMOID, "silu": _lib.GATE_SILU}
MAX_INDEX = 1 << 32

BlockNormGrads = namedtuple("BlockNormGrads", ["x", "residual", "gate", "post_weight", "weight", "scale"])


def _numbers(what, p, seed, index, device):
    """(p, seed, address of the seed or None, index) of dropout for the C ABI"""
    p, index = float(p), int(index)
    if not 0.0 <= p <= 1.0 - 2.0 ** -16:
        raise ValueError(f"{what}: p must be from 0 to 1 - 2^-16, got {p}")
    if not 0 <= index < MAX_INDEX:
        raise ValueError(f"{what}: index must be from 0 to 2^32 - 1, got {index}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise TypeError(f"{what}: a seed on the device must be an int64 tensor of one element")
        check_same(what, "seed", seed, device)
        return p, 0, seed.data_ptr(), index
    if seed is None:
        if p > 0.0:
            raise ValueError(f"{what}: dropout needs a seed")
        seed = 0
    return p, int(seed) & (1 << 64) - 1, None, index


def _dropout(x, p, number, at, index):
    D = x.shape[-1] if x.dim() else 1
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    if x.numel() == 0:
        return y
    x2 = rows_of(x, D)
    with on(x.device) as stream:
        _lib.check(_lib.lib().spanqr_dropout(TYPES[x.dtype], x2.shape[0], D, x2.data_ptr(), x2.stride(0), p, number, at, index,
                                             y.data_ptr(), stream))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, index):
        ctx.how = p, index
        ctx.number = None if isinstance(seed, torch.Tensor) else seed
        if ctx.number is None and seed is not None:
            ctx.save_for_backward(seed)   # (changed in place before the backward pass it would give another mask)
        return _dropout(x, *_numbers("dropout", p, seed, index, x.device))

    @staticmethod
    def backward(ctx, dy):
        p, index = ctx.how
        seed = ctx.saved_tensors[0] if ctx.saved_tensors else ctx.number
        return dropout(dy, p, seed, index), None, None, None


def dropout(x, p, seed=None, index=0):
    """x with a share p of its elements set to 0 and the others divided by 1 - p. x: float32, bfloat16 or float16 [..., D] on a
    ROCm device, any strides; p from 0 to 1 - 2^-16, rounded to a multiple of 2^-16 (and so is the divisor's). What is
    dropped is 0 also where x is infinite or NaN.

    Nothing is kept of the mask: whether element (row, column) of x as [rows, D] is dropped follows from seed, index, row and
    column by a counter-based generator (Philox-4x32-10), whatever x's type and strides. The same call on the gradient
    is the backward pass. seed: a whole number (its low 64 bits), or an int64 tensor of one element on x's device, which a
    captured step can change between replays; needed where p > 0. index, 0 to 2^32 - 1: which of the step's
    dropouts this is, so that one seed serves them all.

    Differentiable in x any number of times."""
    no_tangents("dropout", x)
    check_tensor("dropout", "x", x)
    numbers = _numbers("dropout", p, seed, index, x.device)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dropout.apply(x, p, seed, index)
    return _dropout(x, *numbers)


def _check(what, x, weights, gate, gate_act, scale):
    check_tensor(what, "x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: x must be [..., D] with D >= 1, got {list(x.shape)}")
    kind = None
    for name, w in weights:
        if w is None:
            continue
        if not like(w, x, x.shape[-1:]):
            check_tensor(what, name, w)
            check_same(what, name, w, x.device, (x.shape[-1],))
            if w.dtype != x.dtype and w.dtype != torch.float32:
                raise TypeError(f"{what}: {name} must be float32 or x's type {x.dtype}, got {w.dtype}")
        if kind is not None and w.dtype != kind:
            raise TypeError(f"{what}: post_weight and weight must be of one type, got {kind} and {w.dtype}")
        kind = w.dtype
    if gate_act not in GATES:
        raise ValueError(f"{what}: gate_act must be None, 'sigmoid' or 'silu', got {gate_act!r}")
    if gate is not None:
        check_like(what, "gate", gate, x, x.shape)
    if isinstance(scale, torch.Tensor):
        check_tensor(what, "scale", scale, (torch.float32,))
        check_same(what, "scale", scale, x.device)
        if scale.numel() != 1:
            raise ValueError(f"{what}: scale must have one element")
    return TYPES[x.dtype] if kind is None else TYPES[kind]


def _scale(scale):
    """(number, address or None) for the C ABI"""
    return (0.0, scale.data_ptr()) if isinstance(scale, torch.Tensor) else (float(scale), None)


def _at(t):
    return None if t is None else t.data_ptr()


def _ld(t):
    return 0 if t is None else t.stride(0)


def _dense(w):
    return None if w is None else w.contiguous()


def _rows(t, D):
    return None if t is None else rows_of(t, D)


def _forward(x, residual, post_weight, weight, wtype, gate, gate_act, scale, numbers, eps):
    D, dev = x.shape[-1], x.device
    h = torch.empty_like(x, memory_format=torch.contiguous_format)
    y = torch.empty_like(h)
    x2, r2, g2 = rows_of(x, D), rows_of(residual, D), _rows(gate, D)
    post_weight, weight = _dense(post_weight), _dense(weight)
    number, at = _scale(scale)
    with on(dev) as stream:
        _lib.check(_lib.lib().spanqr_block_norm(
            TYPES[x.dtype], wtype, GATES[gate_act], x2.shape[0], D, x2.data_ptr(), x2.stride(0), r2.data_ptr(), r2.stride(0),
            _at(g2), _ld(g2), _at(post_weight), _at(weight), float(eps), number, at, *numbers, h.data_ptr(), y.data_ptr(),
            stream))
    return y, h


def _backward(dy, dh, x, h, post_weight, weight, wtype, gate, gate_act, scale, p, seed, index, eps, need_weights, need_scale):
    D, dev = x.shape[-1], x.device
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dr = torch.empty_like(dx)
    dg = None if gate is None else torch.empty_like(dx)
    dys, dhs, x2, h2, g2 = _rows(dy, D), _rows(dh, D), rows_of(x, D), rows_of(h, D), _rows(gate, D)
    post_weight, weight = _dense(post_weight), _dense(weight)
    dw1 = torch.empty_like(post_weight) if post_weight is not None and need_weights else None
    dw2 = torch.empty_like(weight) if weight is not None and need_weights else None
    da = torch.empty((), dtype=torch.float32, device=dev) if need_scale else None
    number, at = _scale(scale)
    numbers = _numbers("block_norm_backward", p, seed, index, dev)
    lib, t, nbytes, ws = _lib.lib(), TYPES[x.dtype], 0, None
    with on(dev) as stream:
        if dw1 is not None or dw2 is not None or da is not None:
            nbytes = lib.spanqr_block_norm_backward_workspace(x2.shape[0], D)
            if nbytes < 0:
                _lib.check(nbytes)
            ws = workspace(nbytes, dev)
        _lib.check(lib.spanqr_block_norm_backward(
            t, wtype, GATES[gate_act], x2.shape[0], D, _at(dys), _ld(dys), _at(dhs), _ld(dhs), x2.data_ptr(), x2.stride(0),
            h2.data_ptr(), h2.stride(0), _at(g2), _ld(g2), _at(post_weight), _at(weight), float(eps), number, at, *numbers,
            dx.data_ptr(), dr.data_ptr(), _at(dg), _at(dw1), _at(dw2), _at(da), _at(ws), nbytes, stream))
    return BlockNormGrads(dx, dr, dg, dw1, dw2, da)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, post_weight, weight, gate, scale, wtype, gate_act, p, seed, index, eps):
        y, h = _forward(x, residual, post_weight, weight, wtype, gate, gate_act, scale,
                        _numbers("block_norm", p, seed, index, x.device), eps)
        ctx.scale, ctx.seed = (None if isinstance(v, torch.Tensor) else v for v in (scale, seed))
        ctx.save_for_backward(x, h, post_weight, weight, gate, scale if ctx.scale is None else None,
                              seed if ctx.seed is None else None)
        ctx.how = wtype, gate_act, p, index, eps
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        x, h, post_weight, weight, gate, scale, seed = ctx.saved_tensors
        wtype, gate_act, p, index, eps = ctx.how
        need = ctx.needs_input_grad
        g = _backward(dy, dh, x, h, post_weight, weight, wtype, gate, gate_act, ctx.scale if scale is None else scale, p,
                      ctx.seed if seed is None else seed, index, eps, need[2] or need[3], need[5])
        formed_from = [t for t in (x, h, post_weight, weight, gate, scale, dy, dh) if t is not None]
        out = [once("block_norm", d, *formed_from) for d in g[:5]]
        da = None if g.scale is None else once("block_norm", g.scale.view(scale.shape), *formed_from)
        dx, dr, dg, dw1, dw2 = out
        return dx, dr, dw1, dw2, dg, da, None, None, None, None, None, None


def block_norm(x, residual, post_weight=None, weight=None, gate=None, gate_act="silu", scale=1.0, p=0.0, seed=None, index=0,
               eps=1e-6):
    """(y, h): what a block gives, on its way to the stream and to the next block, over the last axis,

        t = norm(x) * post_weight * act(gate),   h = residual + scale * dropout(t, p),   y = norm(h) * weight

    with norm(v) = v / sqrt(mean(v^2) + eps); h, the stream to go on with, is rounded to x's type and normed as rounded. x:
    float32, bfloat16 or float16 [..., D] on a ROCm device, any strides; residual and gate (or None: no gate) of x's shape
    and type; post_weight and weight [D] of x's type or float32, both of one type, or None for 1. gate_act: "silu",
    "sigmoid", or None for the gate as it is. scale: a number, or a float32 tensor of one element on the device. p, seed and
    index: as in dropout, (row, column) being x's as [rows, D]; p = 0 drops nothing and needs no seed. Sums are float32.

    Differentiable in x, residual, the weights, gate and a scale on the device, once (gradients of the gradients raise
    RuntimeError)."""
    no_tangents("block_norm", x, residual, post_weight, weight, gate, scale)
    wtype = _check("block_norm", x, (("post_weight", post_weight), ("weight", weight)), gate, gate_act, scale)
    check_like("block_norm", "residual", residual, x, x.shape)
    numbers = _numbers("block_norm", p, seed, index, x.device)
    if torch.is_grad_enabled():
        inputs = (x, residual, post_weight, weight, gate, scale)
        if any(isinstance(t, torch.Tensor) and t.requires_grad for t in inputs):
            return _BlockNorm.apply(*inputs, wtype, gate_act, p, seed, index, eps)
    return _forward(x, residual, post_weight, weight, wtype, gate, gate_act, scale, numbers, eps)


def block_norm_backward(dy, dh, x, h, post_weight=None, weight=None, gate=None, gate_act="silu", scale=1.0, p=0.0, seed=None,
                        index=0, eps=1e-6, need_weights=True, need_scale=None):
    """The gradients of block_norm from those of y and of h (dh: what reaches the stream behind it; either may be None for 0),
    with x and gate as they went in, h as it came out, and the other arguments as they were: a named tuple of x, residual,
    gate, post_weight, weight and scale, None where there is no such input, or for the weights with need_weights=False.
    scale's (a float32 tensor without axes) is formed where scale is a tensor, or as need_scale says. None of them
    carries a gradient."""
    what = "block_norm_backward"
    no_tangents(what, dy, dh, x, h, post_weight, weight, gate, scale)
    wtype = _check(what, x, (("post_weight", post_weight), ("weight", weight)), gate, gate_act, scale)
    check_like(what, "h", h, x, x.shape)
    for name, t in (("dy", dy), ("dh", dh)):
        if t is not None:
            check_like(what, name, t, x, x.shape)
    if need_scale is None:
        need_scale = isinstance(scale, torch.Tensor)
    with torch.no_grad():
        return _backward(dy, dh, x, h, post_weight, weight, wtype, gate, gate_act, scale, p, seed, index, eps, need_weights,
                         need_scale)
