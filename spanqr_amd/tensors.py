"""What the training operators (loss.py, norm.py, clip.py) share: types of the C ABI, checks of tensors, and the device
and stream a call runs on."""
import contextlib

import torch
from torch.autograd import forward_ad

from . import _lib

TYPES = {torch.float32: _lib.FP32, torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}


def check_tensor(what, name, t, dtypes=tuple(TYPES)):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what}: {name} must be a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{what}: {name} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {t.dtype}")
    if t.device.type != "cuda":
        raise TypeError(f"{what}: {name} must be on a GPU (ROCm device); there is no CPU implementation")


def check_same(what, name, t, device, shape=None, dtype=None):
    if t.device != device:
        raise ValueError(f"{what}: {name} is on {t.device}, not on {device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} must be {list(shape)}, got {list(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what}: {name} must be {str(dtype)[6:]}, got {t.dtype}")


def like(t, x, shape):
    """whether t has this shape, and the type and device of x, which is checked: the usual case in one short look"""
    return isinstance(t, torch.Tensor) and t.dtype is x.dtype and t.shape == shape and t.get_device() == x.get_device()


def check_like(what, name, t, x, shape):
    if not like(t, x, shape):
        check_tensor(what, name, t)
        check_same(what, name, t, x.device, shape, x.dtype)


def no_tangents(what, *ts):
    """Refuses tensors with a tangent of forward-mode differentiation, which the kernels would leave behind. Outside of it
    (no dual level) nothing is looked at."""
    if forward_ad._current_level < 0:
        return
    for t in ts:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what}: forward-mode differentiation is not implemented")


def rows_of(t, D):
    """t [..., D] as [rows, D] with neighbouring elements in a row; copied only where no such view exists (or rows
    overlap)"""
    if t.dim() != 2:
        t = t.reshape(-1, D)
    if (t.stride(1) != 1 and D > 1) or (t.stride(0) < D and t.shape[0] > 1):
        t = t.contiguous()
    return t


class _Once(torch.autograd.Function):
    """a gradient as it is, behind what it was formed from: its own gradient is refused"""

    @staticmethod
    def forward(ctx, what, grad, *formed_from):
        ctx.what = what
        ctx.mark_dirty(grad)
        return grad

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError(f"{ctx.what}: its gradients cannot be differentiated again")


def once(what, grad, *formed_from):
    """grad as a backward pass returns it. Where that pass records (create_graph) the kernels' result would look like a
    constant, and a function of it would train without its share: it depends on formed_from, and says so when asked."""
    return grad if grad is None or not torch.is_grad_enabled() else _Once.apply(what, grad, *formed_from)


# the current stream's handle by the device's index: what torch.cuda.current_stream(device).cuda_stream gives, without
# the stream object around it (0.1 us instead of 1.9)
_stream = torch._C._cuda_getCurrentRawStream


@contextlib.contextmanager
def _other_device(device):
    with torch.cuda.device(device):
        yield _stream(device.index)


class _Here:
    """`with` on the current device: the stream alone"""
    __slots__ = ("stream",)

    def __init__(self, stream):
        self.stream = stream

    def __enter__(self):
        return self.stream

    def __exit__(self, *exc):
        return False


def on(device):
    """`with on(device) as stream`: the call's current stream on `device`, with that device current"""
    if device.index == torch.cuda.current_device():
        return _Here(_stream(device.index))
    return _other_device(device)


def workspace(nbytes, device):
    """from torch's caching allocator: it may be freed while the call's work is pending on the current stream"""
    return torch.empty(nbytes, dtype=torch.uint8, device=device)
