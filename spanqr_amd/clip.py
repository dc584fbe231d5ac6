"""The norm over many tensors and clipping by it, through the native library (csrc/clip.hip): what a training step does
with its gradients before the optimizer forms the X that orth takes. No counterpart in the reference.
"""
from array import array

import torch

from . import _lib
from .tensors import TYPES, check_same, check_tensor, no_tangents, on, workspace


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


# (called through map: for hundreds of tensors a third less time than a method call each)
_device_of, _dtype_of = torch.Tensor.get_device, torch.Tensor.dtype.__get__


def _tensors(what, name, ts, device=None):
    """ts as a list of tensors of the three types on one GPU, that device, and the tensors' types for the C ABI"""
    ts = [ts] if isinstance(ts, torch.Tensor) else list(ts)
    no_tangents(what, *ts)
    if not ts:
        return ts, device or torch.device("cuda", torch.cuda.current_device()), array("i")
    first = ts[0]
    try:   # hundreds of tensors: what is right is seen in one go, and only what is wrong is looked for
        dev = first.device if device is None else device
        if dev.type == "cuda" and set(map(_device_of, ts)) == {dev.index}:
            kinds = set(map(_dtype_of, ts))
            if len(kinds) == 1:   # as a rule
                return ts, dev, array("i", [TYPES[kinds.pop()]]) * len(ts)
            return ts, dev, _types(ts)
    except (AttributeError, KeyError, TypeError):   # not a tensor, or of another type
        pass
    for t in ts:
        check_tensor(what, name, t)
        check_same(what, name, t, device or first.device)
    return ts, first.device, _types(ts)


def _contiguous(ts):
    return all(map(torch.Tensor.is_contiguous, ts))


def _pointers(ts):
    return array("Q", [t.data_ptr() for t in ts])


def _types(ts):
    return array("i", [TYPES[t.dtype] for t in ts])


def _sizes(ts):
    return array("q", [t.numel() for t in ts])


def _at(values):
    return values.buffer_info()[0]


def grad_norm(grads):
    """sqrt of the sum of squares over all tensors of a list (or of one tensor): float32, bfloat16 and float16 mixed, of
    any shapes and strides, on one ROCm device. A float32 tensor without axes on that device, no host synchronisation;
    squares and sums in float64. An empty list gives 0. The norm carries no gradient, also of tensors that require one."""
    ts, dev, types = _tensors("grad_norm", "every gradient", grads)
    if not _contiguous(ts):
        ts = [t if _dense(t) else t.contiguous() for t in ts]
    n = len(ts)
    at, numel = _pointers(ts), _sizes(ts)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    lib = _lib.lib()
    with on(dev) as stream:
        nbytes = lib.spanqr_grad_norm_workspace(n)
        ws = workspace(nbytes, dev)
        _lib.check(lib.spanqr_grad_norm(n, _at(at), _at(numel), _at(types), norm.data_ptr(), ws.data_ptr(), nbytes, stream))
    return norm


def _in_rows(grads, out, dev):
    """(src, dst, back) where some tensor is strided: pairs that lie in one order, and what is copied back into out
    afterwards"""
    src, dst, back = [], [], []
    for g, o in zip(grads, out):
        if any(s == 0 and n > 1 for s, n in zip(o.stride(), o.shape)):
            raise ValueError("clip_grad_norm: a tensor to write to has elements that share memory (an expanded tensor)")
        if g.stride() == o.stride() and _dense(g):
            src.append(g)
            dst.append(o)
            continue
        src.append(g.contiguous())
        if o.is_contiguous():
            dst.append(o)
        else:
            dst.append(src[-1] if o.dtype == g.dtype and src[-1] is not g else
                       torch.empty(o.shape, dtype=o.dtype, device=dev))
            back.append((o, dst[-1]))
    return src, dst, back


def clip_grad_norm(grads, max_norm, out=None):
    """Scales the gradients by min(1, max_norm / norm), norm = grad_norm(grads), and returns the norm (before clipping;
    float32 on the device, no host synchronisation). In place; or, with out (a list of tensors of the same shapes, of
    any of the three types), into out, the gradients left as they are: float32 copies of 16-bit gradients in the same
    pass, for an optimizer that works in float32. In place a norm within max_norm writes nothing.

    Each tensor to write to is listed once (a shared parameter's gradient, too): two that start at the same address raise
    ValueError. out may share no memory with the gradients, other than out[i] being grads[i]. A NaN gradient makes
    every result NaN, an infinite one makes the finite ones 0: look at the norm before the step. Neither the norm nor what is
    written carries a gradient."""
    grads, dev, types = _tensors("clip_grad_norm", "every gradient", grads)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grad_norm: max_norm must not be negative, got {max_norm}")
    if out is None:
        out, out_types = grads, types
    else:
        out, _, out_types = _tensors("clip_grad_norm", "every tensor of out", out, dev)
        if len(out) != len(grads) or not all(map(torch.Tensor.is_same_size, grads, out)):
            if len(out) != len(grads):
                raise ValueError(f"clip_grad_norm: {len(grads)} gradients but {len(out)} tensors in out")
            for g, o in zip(grads, out):
                check_same("clip_grad_norm", "a tensor of out", o, dev, g.shape)
    back = ()
    src, dst = grads, out
    if not (_contiguous(grads) and (out is grads or _contiguous(out))):
        src, dst, back = _in_rows(grads, out, dev)
    n = len(src)
    at, numel = _pointers(src), _sizes(src)
    to = at if dst is src else _pointers(dst)
    if len(set(to)) < n:   # (empty tensors have no address)
        full = [p for p, k in zip(to, numel) if k]
        if len(set(full)) < len(full):
            raise ValueError("clip_grad_norm: two of the tensors to write to lie in the same memory")
    norm = torch.empty((), dtype=torch.float32, device=dev)
    lib = _lib.lib()
    with on(dev) as stream:
        nbytes = lib.spanqr_grad_norm_workspace(n)
        ws = workspace(nbytes, dev)
        _lib.check(lib.spanqr_clip_grad_norm(n, _at(at), _at(numel), _at(types), _at(to), _at(out_types), max_norm,
                                             norm.data_ptr(), ws.data_ptr(), nbytes, stream))
    # written behind autograd's back, which has to notice if it keeps one of them (whether the norm was within max_norm is
    # not known here)
    torch.autograd.graph.increment_version(out)
    if back:
        with torch.no_grad():   # as the others are written
            for o, copy in back:
                o.copy_(copy)
    return norm
