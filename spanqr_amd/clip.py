"""The norm over many tensors and clipping by it, through the native library (csrc/clip.hip): what a training step does
with its gradients before the optimizer forms the X that orth takes. No counterpart in the reference.
"""
import ctypes

import torch

from . import _lib
from .tensors import TYPES, check_same, check_tensor, on, workspace


def _dense(t):
    """whether t's elements fill one stretch of memory, each once, in whatever order"""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _check(what, grads):
    if isinstance(grads, torch.Tensor):
        grads = [grads]
    grads = list(grads)
    for g in grads:
        check_tensor(what, "every gradient", g)
        check_same(what, "a gradient", g, grads[0].device)
    return grads


def _table(ts):
    """host arrays of the tensors' addresses and of their types"""
    n = len(ts)
    return ((ctypes.c_void_p * n)(*[t.data_ptr() for t in ts]), (ctypes.c_int * n)(*[TYPES[t.dtype] for t in ts]))


def _norm_device(grads):
    return grads[0].device if grads else torch.device("cuda", torch.cuda.current_device())


def grad_norm(grads):
    """sqrt of the sum of squares over all tensors of a list (or of one tensor): float32, bfloat16 and float16 mixed, of
    any shapes and strides, on one ROCm device. A float32 tensor without axes on that device, no host synchronisation;
    squares and sums in float64. An empty list gives 0."""
    grads = _check("grad_norm", grads)
    dev = _norm_device(grads)
    ts = [g if _dense(g) else g.contiguous() for g in grads]
    n = len(ts)
    at, types = _table(ts)
    numel = (ctypes.c_long * n)(*[t.numel() for t in ts])
    norm = torch.empty((), dtype=torch.float32, device=dev)
    with on(dev) as stream:
        nbytes = _lib.lib().spanqr_grad_norm_workspace(n)
        ws = workspace(nbytes, dev)
        _lib.check(_lib.lib().spanqr_grad_norm(n, at, numel, types, norm.data_ptr(), ws.data_ptr(), nbytes, stream))
    return norm


def clip_grad_norm(grads, max_norm, out=None):
    """Scales the gradients by min(1, max_norm / norm), norm = grad_norm(grads), and returns the norm (before clipping;
    float32 on the device, no host synchronisation). In place; or, with out (a list of tensors of the same shapes, of
    any of the three types), into out, the gradients left as they are: float32 copies of 16-bit gradients in the same
    pass, for an optimizer that works in float32. In place a norm within max_norm writes nothing.

    A NaN norm makes every result NaN, an infinite norm makes finite gradients 0: look at the norm before the step. out
    may share no memory with the gradients, other than out[i] being grads[i]."""
    grads = _check("clip_grad_norm", grads)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grad_norm: max_norm must not be negative, got {max_norm}")
    dev = _norm_device(grads)
    if out is None:
        out = grads
    else:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(out) != len(grads):
            raise ValueError(f"clip_grad_norm: {len(grads)} gradients but {len(out)} tensors in out")
        for g, o in zip(grads, out):
            check_tensor("clip_grad_norm", "every tensor of out", o)
            check_same("clip_grad_norm", "a tensor of out", o, dev, g.shape)
    src, dst, back = [], [], []
    for g, o in zip(grads, out):
        if any(s == 0 and n > 1 for s, n in zip(o.stride(), o.shape)):
            raise ValueError("clip_grad_norm: a tensor to write to has elements that share memory (an expanded tensor)")
        same = g.stride() == o.stride()
        if same and _dense(g):
            src.append(g)
            dst.append(o)
            continue
        # strided views, or two different orders: through a copy that lies in rows
        src.append(g.contiguous())
        if o.is_contiguous():
            dst.append(o)
        else:
            dst.append(src[-1] if o.dtype == g.dtype and src[-1] is not g else
                       torch.empty(o.shape, dtype=o.dtype, device=dev))
            back.append((o, dst[-1]))
    n = len(src)
    at, types = _table(src)
    to, out_types = _table(dst)
    numel = (ctypes.c_long * n)(*[t.numel() for t in src])
    norm = torch.empty((), dtype=torch.float32, device=dev)
    with on(dev) as stream:
        nbytes = _lib.lib().spanqr_grad_norm_workspace(n)
        ws = workspace(nbytes, dev)
        _lib.check(_lib.lib().spanqr_clip_grad_norm(n, at, numel, types, to, out_types, max_norm, norm.data_ptr(),
                                                    ws.data_ptr(), nbytes, stream))
    for o, copy in back:
        o.copy_(copy)
    return norm
