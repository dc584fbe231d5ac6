"""Softmax cross entropy over a large vocabulary from the hidden states and the head's weights, without keeping the
logits, with its gradients, through the native library (csrc/loss.hip). No counterpart in the reference; it is where the
gradients begin that end in the optimizer's orth.
"""
import torch

from . import _lib
from .tensors import TYPES, check_same, check_tensor, no_tangents, on, once, workspace

IGNORE_INDEX = -100
MAX_WORKSPACE = 4 << 30   # bytes: 16-bit exponentials of 15000 tokens over 128000 columns, with their statistics
MAX_STRIDE = 1 << 22
REDUCTIONS = {"none": _lib.REDUCE_NONE, "sum": _lib.REDUCE_SUM, "mean": _lib.REDUCE_MEAN}


def _rows(t):
    """rows of neighbouring elements, apart from each other but not further than the library's offsets reach"""
    if (t.stride(1) != 1 and t.shape[1] > 1) or (not t.shape[1] <= t.stride(0) <= MAX_STRIDE and t.shape[0] > 1):
        t = t.contiguous()
    return t


def _check(what, x, weight, target, reduction, row_weight, grad_scale=None):
    no_tangents(what, x, weight, row_weight, grad_scale)
    check_tensor(what, "x", x, (torch.bfloat16, torch.float16))
    check_tensor(what, "weight", weight, (torch.bfloat16, torch.float16))
    if x.dim() != 2 or weight.dim() != 2:
        raise ValueError(f"{what}: x must be [N, H] and weight [V, H], got {list(x.shape)} and {list(weight.shape)}")
    H, V = x.shape[1], weight.shape[0]
    if H < 1 or V < 1:
        raise ValueError(f"{what}: H = {H} and V = {V} must be at least 1")
    check_same(what, "weight", weight, x.device, (V, H), x.dtype)
    if not isinstance(target, torch.Tensor) or target.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: target must be an int64 or int32 tensor")
    check_same(what, "target", target, x.device, (x.shape[0],))
    if reduction not in REDUCTIONS:
        raise ValueError(f"{what}: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    if row_weight is not None:
        check_tensor(what, "row_weight", row_weight, (torch.float32,))
        check_same(what, "row_weight", row_weight, x.device, (x.shape[0],))


def _run(x, weight, target, reduction, ignore_index, row_weight, grad_scale, need_dx, need_dw, max_workspace):
    x, weight = _rows(x.detach()), _rows(weight.detach())
    (N, H), V, dev = x.shape, weight.shape[0], x.device
    target = target.to(torch.int64).contiguous()
    if row_weight is not None:
        row_weight = row_weight.contiguous()
    loss = torch.empty((N,) if reduction == "none" else (), dtype=torch.float32, device=dev)
    dx = torch.empty(N, H, dtype=x.dtype, device=dev) if need_dx else None
    dw = torch.empty(V, H, dtype=x.dtype, device=dev) if need_dw else None
    t, grads = TYPES[x.dtype], int(need_dx) + 2 * int(need_dw)
    if (x.data_ptr() | weight.data_ptr() | 2 * (x.stride(0) if N > 1 else 0) | 2 * (weight.stride(0) if V > 1 else 0)) % 16:
        grads += 4   # rows that do not start on 16 bytes are copied once
    with on(dev) as stream:
        nbytes = _lib.lib().spanqr_linear_cross_entropy_workspace(t, N, H, V, grads, int(max_workspace))
        if nbytes < 0:
            _lib.check(nbytes)
        ws = workspace(nbytes, dev)
        _lib.check(_lib.lib().spanqr_linear_cross_entropy(
            t, REDUCTIONS[reduction], N, H, V, x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0),
            target.data_ptr(), int(ignore_index), None if row_weight is None else row_weight.data_ptr(),
            None if grad_scale is None else grad_scale.data_ptr(), loss.data_ptr(), None,
            None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(), ws.data_ptr(), nbytes, stream))
    return loss, dx, dw


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, reduction, ignore_index, max_workspace):
        loss, _, _ = _run(x, weight, target, reduction, ignore_index, None, None, False, False, max_workspace)
        ctx.save_for_backward(x, weight, target)
        ctx.how = reduction, ignore_index, max_workspace
        return loss

    @staticmethod
    def backward(ctx, g):
        x, weight, target = ctx.saved_tensors
        reduction, ignore_index, max_workspace = ctx.how
        f = g.detach().to(torch.float32)
        _, dx, dw = _run(x, weight, target, reduction, ignore_index, f.contiguous() if reduction == "none" else None,
                         None if reduction == "none" else f, ctx.needs_input_grad[0], ctx.needs_input_grad[1],
                         max_workspace)
        dx, dw = (once("linear_cross_entropy", d, x, weight, g) for d in (dx, dw))
        return dx, dw, None, None, None, None


def linear_cross_entropy(x, weight, target, reduction="mean", ignore_index=IGNORE_INDEX, max_workspace=MAX_WORKSPACE):
    """Cross entropy of softmax(x weight^T) against target: x [N, H] and weight [V, H] bfloat16 or float16 on a ROCm
    device, target [N] int64 or int32. float32: the mean over the tokens whose target is not ignore_index (0 if there are
    none), the sum, or ("none") each token's loss [N], 0 where ignored. The logits are not kept. A target that is neither a
    column nor ignore_index gives NaN.

    Differentiable in x and weight, once (gradients of the gradients raise RuntimeError); the backward pass forms the
    logits again with the incoming gradient at hand. A training step that wants the gradients at once takes
    linear_cross_entropy_grad, which forms the logits once. max_workspace: bytes of scratch memory that bound how many
    tokens are taken at a time."""
    _check("linear_cross_entropy", x, weight, target, reduction, None)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _LinearCrossEntropy.apply(x, weight, target, reduction, ignore_index, max_workspace)
    return _run(x, weight, target, reduction, ignore_index, None, None, False, False, max_workspace)[0]


def linear_cross_entropy_grad(x, weight, target, reduction="mean", ignore_index=IGNORE_INDEX, row_weight=None,
                              grad_scale=None, need_dx=True, need_dw=True, max_workspace=MAX_WORKSPACE):
    """(loss, dx, dw): linear_cross_entropy and its gradients in one pass, in x's type. row_weight [N] float32 multiplies
    each token's loss (not the count that the mean is over). grad_scale (a number, or a float32 tensor of one element on
    the device: a loss scale) multiplies the gradients before they are rounded, not the loss. With reduction "none" the
    gradients are of the sum. dx or dw is None with need_dx=False or need_dw=False. None of them carries a gradient.

    Sums are float32. Above 32 tokens each element of softmax - onehot is rounded to x's type twice on its way into the
    gradients: their error is 1.0 to 1.3 times that of a float32 result that is rounded once, 1.7 times at most. x of ignored
    tokens has to be finite for dw, where it is multiplied by 0."""
    _check("linear_cross_entropy_grad", x, weight, target, reduction, row_weight, grad_scale)
    if grad_scale is not None:
        if not isinstance(grad_scale, torch.Tensor):
            grad_scale = torch.full((), float(grad_scale), dtype=torch.float32, device=x.device)
        check_tensor("linear_cross_entropy_grad", "grad_scale", grad_scale, (torch.float32,))
        check_same("linear_cross_entropy_grad", "grad_scale", grad_scale, x.device)
        if grad_scale.numel() != 1:
            raise ValueError("linear_cross_entropy_grad: grad_scale must have one element")
    return _run(x, weight, target, reduction, ignore_index, row_weight, grad_scale, need_dx, need_dw, max_workspace)
