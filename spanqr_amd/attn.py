"""Softmax attention with heads that share keys and values, for padded batches and packed sequences, and its gradient, which
makes the probabilities again, through the native library (csrc/attention.hip). No counterpart in the reference; its
projections are among the layers that the optimizer keeps orthonormal with orth.
"""
import functools
from array import array

import torch

from . import _lib
from .tensors import TYPES, check_like, check_same, check_tensor, like, no_tangents, on, once, workspace

MAX_STRIDE = 1 << 24   # of rows, and of q's, the result's and its gradient's heads, in elements
MAX_HEAD = 128
MOST = 1 << 40         # more keys or rows than there are say the same, and this fits into the C ABI's numbers


def _heads(t, keys=False):
    """(t, its strides {batch, row, head}): neighbouring elements of a head, every head's row on 16 bytes, and strides that the
    library's offsets reach (keys: k's and v's heads may lie any way apart); as it lies, or copied"""
    s = t.stride()
    if s[-1] != 1 or (s[0] | s[-2] | s[-3]) & 7 or (s[-2] >= MAX_STRIDE and not keys) or s[-3] >= MAX_STRIDE:
        far = t.dim() - 4, t.dim() - 2 if keys else None
        if not ((s[-1] == 1 or t.shape[-1] == 1) and all(
                n == 1 or (v % 8 == 0 and (v < MAX_STRIDE or i in far)) for i, (n, v) in enumerate(zip(t.shape[:-1], s)))):
            t = t.contiguous()
            s = t.stride()
        s = tuple(0 if n == 1 else v for n, v in zip(t.shape, s))   # (axes of one element have any)
    if t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        s = t.stride()
    return t, (s[:3] if t.dim() == 4 else (0, *s[:2]))


def _check(what, q, k, v, causal, window, scale, q_starts, k_starts, max_q, max_k, k_lens):
    """the shape as the C ABI takes it: B, key heads, group, D, Tq, Tk; and the other arguments settled"""
    check_tensor(what, "q", q, (torch.bfloat16, torch.float16))
    packed = q_starts is not None
    if not packed and (k_starts is not None or max_q is not None or max_k is not None):
        raise ValueError(f"{what}: k_starts, max_q and max_k belong to packed sequences, which need q_starts")
    if packed and k_lens is not None:
        raise ValueError(f"{what}: packed sequences have their lengths from k_starts, not from k_lens")
    axes = 3 if packed else 4
    for name, t in (("q", q), ("k", k), ("v", v)):
        check_tensor(what, name, t, (torch.bfloat16, torch.float16))
        if t.dim() != axes:
            raise ValueError(f"{what}: {name} must be " + ("[rows, heads, D] with q_starts" if packed else "[B, S, heads, D]") +
                             f", got {list(t.shape)}")
    *lead, Tq, heads, D = q.shape
    Tk, key_heads = k.shape[-3:-1]
    if D < 8 or D > MAX_HEAD or D % 8:
        raise ValueError(f"{what}: D must be a multiple of 8 from 8 to {MAX_HEAD}, got {D}")
    if heads < 1 or key_heads < 1 or heads % key_heads:
        raise ValueError(f"{what}: q's {heads} heads must be a multiple of k's {key_heads}, one at least")
    key_shape = (*lead, Tk, key_heads, D)
    if not (like(k, q, key_shape) and like(v, q, key_shape)):
        check_same(what, "k", k, q.device, key_shape, q.dtype)
        check_same(what, "v", v, q.device, key_shape, q.dtype)
    if window is not None:
        window = int(window)
        if window < 1 or not causal:
            raise ValueError(f"{what}: a window is at least 1 and needs causal=True, got {window}")
        window = min(window, MOST)
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"{what}: scale must be positive and finite, got {scale}")
    if packed:
        if k_starts is None:
            if Tq != Tk:
                raise ValueError(f"{what}: without k_starts q and k have the same rows, got {Tq} and {Tk}")
            k_starts = q_starts
            max_k = max_q if max_k is None else max_k
        for name, t in (("q_starts", q_starts), ("k_starts", k_starts)):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
                raise TypeError(f"{what}: {name} must be an int32 tensor")
            check_same(what, name, t, q.device)
            if t.dim() != 1 or t.numel() < 1 or t.numel() != q_starts.numel():
                raise ValueError(f"{what}: q_starts and k_starts must be [B + 1], of one length")
        B = q_starts.numel() - 1
        q_starts, k_starts = q_starts.contiguous(), k_starts.contiguous()
    else:
        B = lead[0]
        if k_lens is not None:
            if not isinstance(k_lens, torch.Tensor) or k_lens.dtype != torch.int32:
                raise TypeError(f"{what}: k_lens must be an int32 tensor")
            check_same(what, "k_lens", k_lens, q.device, (B,))
            k_lens = k_lens.contiguous()
    for name, n in (("max_q", max_q), ("max_k", max_k)):
        if n is not None and int(n) < 0:
            raise ValueError(f"{what}: {name} must not be negative, got {n}")
    return (B, key_heads, heads // key_heads, D, Tq, Tk), window or 0, scale, (q_starts, k_starts, k_lens), *(
        min(int(n or 0), MOST) for n in (max_q, max_k))


@functools.lru_cache(maxsize=256)
def _workspace(backward, *sizes):
    """bytes, by sizes alone"""
    lib = _lib.lib()
    nbytes = (lib.spanqr_attention_backward_workspace if backward else lib.spanqr_attention_workspace)(*sizes)
    if nbytes < 0:
        _lib.check(nbytes)
    return nbytes


def _at(t):
    return None if t is None else t.data_ptr()


def _forward(q, k, v, causal, how, need_lse):
    shape, window, scale, (q_starts, k_starts, k_lens), max_q, max_k = how
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if need_lse else None
    (q, qs), (k, ks), (v, vs) = _heads(q), _heads(k, True), _heads(v, True)
    strides = array("q", qs + ks + vs)
    at = strides.buffer_info()[0]
    dev = q.device
    with on(dev) as stream:
        nbytes = _workspace(False, *shape, q_starts is not None, max_q, max_k)
        ws = workspace(nbytes, dev) if nbytes else None
        _lib.check(_lib.lib().spanqr_attention(
            TYPES[q.dtype], *shape, q.data_ptr(), at, k.data_ptr(), at + 24, v.data_ptr(), at + 48, _at(q_starts), _at(k_starts),
            _at(k_lens), max_q, max_k, causal, window, scale, out.data_ptr(), _at(lse), _at(ws), nbytes, stream))
    return out, lse


def _backward(dout, q, k, v, out, lse, causal, how, need_dq, need_dkv):
    shape, window, scale, (q_starts, k_starts, k_lens), max_q, max_k = how
    dev = q.device
    dq = torch.empty(q.shape, dtype=q.dtype, device=dev) if need_dq else None
    dk = torch.empty(k.shape, dtype=q.dtype, device=dev) if need_dkv else None
    dv = torch.empty_like(dk) if need_dkv else None
    (dout, ds), (q, qs), (out, os) = map(_heads, (dout, q, out))
    (k, ks), (v, vs) = _heads(k, True), _heads(v, True)
    strides = array("q", ds + qs + ks + vs + os)
    at = strides.buffer_info()[0]
    lse = lse.contiguous()
    with on(dev) as stream:
        nbytes = _workspace(True, *shape, q_starts is not None, max_q, max_k)
        ws = workspace(nbytes, dev)
        _lib.check(_lib.lib().spanqr_attention_backward(
            TYPES[q.dtype], *shape, dout.data_ptr(), at, q.data_ptr(), at + 24, k.data_ptr(), at + 48, v.data_ptr(), at + 72,
            out.data_ptr(), at + 96, lse.data_ptr(), _at(q_starts), _at(k_starts), _at(k_lens), max_q, max_k, causal, window, scale,
            _at(dq), _at(dk), _at(dv), ws.data_ptr(), nbytes, stream))
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, how):
        out, lse = _forward(q, k, v, causal, how, True)
        shape, window, scale, lengths, max_q, max_k = how
        ctx.save_for_backward(q, k, v, out, lse, *lengths)
        ctx.how = causal, shape, window, scale, max_q, max_k
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    def backward(ctx, dout, _):
        if dout is None:
            return None, None, None, None, None
        q, k, v, out, lse, *lengths = ctx.saved_tensors
        causal, shape, window, scale, max_q, max_k = ctx.how
        need = ctx.needs_input_grad
        grads = _backward(dout, q, k, v, out, lse, causal, (shape, window, scale, lengths, max_q, max_k), need[0],
                          need[1] or need[2])
        return (*(once("attention", g, q, k, v, dout) for g in grads), None, None)


def attention(q, k, v, causal=False, window=None, scale=None, q_starts=None, k_starts=None, max_q=None, max_k=None,
              return_lse=False, k_lens=None):
    """softmax(scale q k^T) v for each head: q [B, Sq, heads, D], k and v [B, Sk, key heads, D], bfloat16 or float16 on a ROCm
    device, heads a multiple of the key heads (head h reads key head h // (heads / key heads)), D a multiple of 8 up to
    128; scale (positive) is D^-1/2 unless given. Strided tensors, such as the columns of one product, are read as they lie
    where every head's row starts on 16 bytes and rows (of q, heads too) are less than 2^24 elements apart, and copied
    elsewhere. The result has q's shape and is contiguous.

    Query i stands at p = i + Sk - Sq, so that one token's query reads all that is cached. causal: it sees the keys j <= p;
    window: only the last `window` of those. A query that sees no key has the result 0. k_lens: int32 [B] on the device, the
    number of keys that a sequence has of k's Sk (a cache with room); it stands for Sk in all this, and the rows behind are
    not read.

    Packed sequences: q [Tq, heads, D], k and v [Tk, key heads, D], with the sequences' rows end to end: those of sequence b are
    q_starts[b] to q_starts[b + 1] - 1, and k_starts' for the keys (q_starts again where it is not given), int32 [B + 1] on
    the device, ascending. They are read on the device, when the work runs: rows in front of the first sequence and
    behind the last one are not read and have the result 0. max_q and max_k: the longest sequence's rows, as far as
    known; they set how much is launched, and so over how many parts sums go, but nothing else of what comes out. Without them the
    launch goes by all rows and the number of sequences.

    The probabilities are rounded to 16 bits before the product with v; scores, softmax and sums are float32. Within a
    sequence q, k and v have to be finite, also where a mask hides them.

    return_lse: (result, lse), with lse [..., heads] float32 the logarithm of each query's sum of exp(scores), -inf where it sees
    no key; attention_backward takes it. Differentiable in q, k and v, once (gradients of the gradients raise RuntimeError);
    lse carries no gradient."""
    no_tangents("attention", q, k, v)
    causal = bool(causal)
    how = _check("attention", q, k, v, causal, window, scale, q_starts, k_starts, max_q, max_k, k_lens)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _Attention.apply(q, k, v, causal, how)
    else:
        out, lse = _forward(q, k, v, causal, how, return_lse)
    return (out, lse) if return_lse else out


def attention_backward(dout, q, k, v, out, lse, causal=False, window=None, scale=None, q_starts=None, k_starts=None, max_q=None,
                       max_k=None, need_dq=True, need_dkv=True, k_lens=None):
    """(dq, dk, dv): attention's gradients from the gradient dout of its result, with out and lse as it returned them and the
    other arguments as they were. Contiguous, in the inputs' type; rows of no sequence and keys behind k_lens have the gradient 0. dq is None
    with need_dq=False, dk and dv with need_dkv=False. The probabilities are made again from q, k and lse; they, and the
    scores' gradients, are rounded to 16 bits before the products that they go into. The sums over the heads that share
    keys are float32, in a fixed order: a call repeats its bits. None of the gradients carries a gradient."""
    what = "attention_backward"
    no_tangents(what, dout, q, k, v, out, lse)
    causal = bool(causal)
    how = _check(what, q, k, v, causal, window, scale, q_starts, k_starts, max_q, max_k, k_lens)
    check_like(what, "dout", dout, q, q.shape)
    check_like(what, "out", out, q, q.shape)
    check_tensor(what, "lse", lse, (torch.float32,))
    check_same(what, "lse", lse, q.device, q.shape[:-1])
    with torch.no_grad():
        return _backward(dout, q, k, v, out, lse, causal, how, need_dq, need_dkv)
