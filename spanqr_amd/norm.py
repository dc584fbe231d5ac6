"""Root-mean-square norm with the residual's addition, in the model's type or in 8 bits with a scale a row, and its
gradient, through the native library (csrc/norm.hip). No counterpart in the reference; it stands before the products
whose gradients the optimizer that calls orth works on.
"""
import torch

from . import _lib
from .tensors import TYPES, check_like, check_same, check_tensor, like, no_tangents, on, once, rows_of, workspace

QUANT = {None: (_lib.QUANT_NONE, None), "fp8": (_lib.QUANT_FP8, torch.float8_e4m3fn), "int8": (_lib.QUANT_INT8, torch.int8)}


def _check(what, x, weight, *others):
    no_tangents(what, x, weight, *others)
    check_tensor(what, "x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: x must be [..., D] with D >= 1, got {list(x.shape)}")
    if weight is not None and not like(weight, x, x.shape[-1:]):
        check_tensor(what, "weight", weight)
        check_same(what, "weight", weight, x.device, (x.shape[-1],))
        if weight.dtype != x.dtype and weight.dtype != torch.float32:
            raise TypeError(f"{what}: weight must be float32 or x's type {x.dtype}, got {weight.dtype}")


def _forward(x, weight, residual, eps, quant):
    D = x.shape[-1]
    x2 = rows_of(x, D)
    dev = x.device
    code, qtype = QUANT[quant]   # (no type of its own: x's)
    r2 = h = scale = None
    if residual is not None:
        r2 = rows_of(residual, D)
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
    y = torch.empty_like(x, dtype=qtype, memory_format=torch.contiguous_format)
    if code:
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    if weight is not None:
        weight = weight.contiguous()
    t = TYPES[x.dtype]
    with on(dev) as stream:
        _lib.check(_lib.lib().spanqr_rms_norm(
            t, t if weight is None else TYPES[weight.dtype], code, x2.shape[0], D, x2.data_ptr(), x2.stride(0),
            None if r2 is None else r2.data_ptr(), 0 if r2 is None else r2.stride(0),
            None if weight is None else weight.data_ptr(), float(eps), None if h is None else h.data_ptr(),
            y.data_ptr(), None if scale is None else scale.data_ptr(), stream))
    return y, scale, h


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, _, h = _forward(x, weight, residual, eps, None)
        ctx.save_for_backward(x if h is None else h, weight)
        ctx.eps, ctx.residual = eps, residual is not None
        ctx.set_materialize_grads(False)
        return (y, h) if ctx.residual else y

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        if dy is None:                       # only the stream went on
            return dh, None if weight is None else torch.zeros_like(weight), dh if ctx.residual else None, None
        dx, dw = rms_norm_backward(dy, h, weight, ctx.eps, dh, ctx.needs_input_grad[1])
        dx, dw = (once("rms_norm", d, h, weight, dy, dh) for d in (dx, dw))
        return dx, dw, dx if ctx.residual else None, None


def rms_norm(x, weight=None, residual=None, eps=1e-6, quant=None):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last axis, with h = x, or h = x + residual (rounded to x's type,
    and normed as rounded). x: float32, bfloat16 or float16 [..., D] on a ROCm device, any strides; weight [D] of x's
    type or float32, or None for 1; residual of x's shape and type. Sums are float32.

    Returns y; with residual (y, h): h is the stream to go on with. With quant="fp8" (float8_e4m3fn) or "int8" y is 8 bits and
    comes with its scale [...] float32, (y, scale) or (y, scale, h): y * scale is the norm, the scale is max|norm| / 448 or
    / 127 of each row. A row of zeros has scale 0; a row with a NaN has scale NaN.

    Differentiable in x, weight and residual without quant, once (gradients of the gradients raise RuntimeError); with
    quant the result carries no gradient (rms_norm_backward takes the gradient of the unrounded norm, as a
    straight-through step does)."""
    _check("rms_norm", x, weight, residual)
    if quant not in QUANT:
        raise ValueError(f"rms_norm: quant must be None, 'fp8' or 'int8', got {quant!r}")
    if residual is not None:
        check_like("rms_norm", "residual", residual, x, x.shape)
    if quant is None and torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad) or
            (residual is not None and residual.requires_grad)):
        return _RmsNorm.apply(x, weight, residual, eps)
    y, scale, h = _forward(x, weight, residual, eps, quant)
    if quant is None:
        return y if h is None else (y, h)
    return (y, scale) if h is None else (y, scale, h)


def rms_norm_backward(dy, h, weight=None, eps=1e-6, dh=None, need_dw=True):
    """(dx, dw) of rms_norm from the gradient dy of y and the normed stream h (x itself where there was no residual):
    dx is the gradient of x and of the residual alike. dh: the gradient that reaches h on the stream's own way, added to
    dx. dw is None without a weight or with need_dw=False; it has the weight's type. Neither carries a gradient."""
    _check("rms_norm_backward", h, weight, dy, dh)
    D, dev = h.shape[-1], h.device
    check_like("rms_norm_backward", "dy", dy, h, h.shape)
    if dh is not None:
        check_like("rms_norm_backward", "dh", dh, h, h.shape)
        dh = rows_of(dh, D)
    h2, dy = rows_of(h, D), rows_of(dy, D)
    dx = torch.empty_like(h, memory_format=torch.contiguous_format)
    dw = ws = None
    nbytes = 0
    if weight is not None:
        weight = weight.contiguous()
        if need_dw:
            dw = torch.empty_like(weight)
            nbytes = _lib.lib().spanqr_rms_norm_backward_workspace(h2.shape[0], D)
            if nbytes < 0:
                _lib.check(nbytes)
    t = TYPES[h.dtype]
    with on(dev) as stream:
        if nbytes:
            ws = workspace(nbytes, dev)
        _lib.check(_lib.lib().spanqr_rms_norm_backward(
            t, t if weight is None else TYPES[weight.dtype], h2.shape[0], D, dy.data_ptr(), dy.stride(0), h2.data_ptr(),
            h2.stride(0), None if weight is None else weight.data_ptr(), None if dh is None else dh.data_ptr(),
            0 if dh is None else dh.stride(0), float(eps), dx.data_ptr(), None if dw is None else dw.data_ptr(),
            None if ws is None else ws.data_ptr(), nbytes, stream))
    return dx, dw
