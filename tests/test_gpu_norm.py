"""rms_norm and rms_norm_backward against the formulas in 64 bits.

The bounds: u is the type's unit roundoff (2^-8 bfloat16, 2^-11 float16, 2^-24 float32). A thread adds at most 32
squares in a row (longer rows: D / 1024), then a tree and a few partial sums, so a sum of D terms is within C 2^-24 of the sum
of its terms' magnitudes with C = 64 + D / 1024; the root halves a relative error, and the products after it add a few
more roundings. The result's own rounding is u of it, or half the smallest subnormal."""
import math

import pytest
import torch

import spanqr_amd as sp

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}
SIZES = [(1, 1), (3, 2), (5, 7), (17, 8), (70, 9), (33, 64), (100, 127), (41, 128), (9, 129), (6, 511), (3, 512),
         (13, 769), (5, 1024), (7, 1025), (10, 2048), (3, 2049), (300, 4096), (2, 5120), (600, 5120), (3, 8191), (4, 8193),
         (2, 16384), (3, 17408), (2, 32768), (3, 32769), (2, 70001)]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(rows, D, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(rows, D, generator=g, device="cuda")).to(dtype)


def weight_of(D, dtype, seed):
    return (1.0 + 0.3 * make(1, D, torch.float32, seed)[0]).to(dtype)


def c_of(D):
    return 64.0 + D / 1024.0


def reference(h, w, eps):
    """(y, s) in 64 bits"""
    h = h.double()
    s = 1.0 / torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[-1] + eps)
    return h * s * (1.0 if w is None else w.double()), s


def check(what, got, want, bound):
    assert got.shape == want.shape, what
    d = (got.double() - want).abs()
    ok = (d <= bound) | (torch.isnan(got) & torch.isnan(want))
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} outside, worst {float((d / bound).nan_to_num().max()):.3g}"


def check_y(what, y, h, w, eps, dtype):
    want, _ = reference(h, w, eps)
    check(what, y, want, want.abs() * (U[dtype] + (c_of(h.shape[-1]) + 8) * E) + TINY[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", SIZES)
def test_forward(cuda, rows, D, dtype):
    print(f"rms_norm {rows}x{D} {dtype}", flush=True)
    x, r, w = make(rows, D, dtype, 1), make(rows, D, dtype, 2, 3.0), weight_of(D, dtype, 3)
    check_y("y", sp.rms_norm(x, w, eps=1e-5), x, w, 1e-5, dtype)
    y, h = sp.rms_norm(x, w.float(), residual=r)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    check_y("y of the sum", y, h, w.float(), 1e-6, dtype)
    check_y("without weight", sp.rms_norm(x), x, None, 1e-6, dtype)


def steps(v, quant):
    """half the distance of neighbouring 8-bit values around v (v in units of the scale)"""
    if quant == "int8":
        return torch.full_like(v, 0.5)
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))).clamp(max=8.0)   # normal from 2^-6, three bits after the first
    return torch.exp2(e - 4)


def dequantised(q, scale):
    return q.double() * scale.double()[..., None]


@pytest.mark.parametrize("quant", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", SIZES)
def test_8_bits(cuda, rows, D, dtype, quant):
    print(f"rms_norm {quant} {rows}x{D} {dtype}", flush=True)
    x, r, w = make(rows, D, dtype, 4), make(rows, D, dtype, 5), weight_of(D, dtype, 6)
    M = 448.0 if quant == "fp8" else 127.0
    for kw in (dict(), dict(residual=r)):
        got = sp.rms_norm(x, w, quant=quant, **kw)
        q, scale = got[:2]
        assert q.dtype == (torch.float8_e4m3fn if quant == "fp8" else torch.int8) and scale.dtype == torch.float32
        h = got[2] if kw else x
        y, _ = reference(h, w, 1e-6)
        c = (c_of(D) + 8) * E
        amax = y.abs().amax(-1)
        check("scale", scale, amax / M, amax / M * c)
        # a value lies at most half a step from its code; the arithmetic before it is c of the value off
        v = y / scale.double()[:, None]
        off = (q.double() - v).abs()
        assert bool((off <= steps(v, quant) * (1 + 1e-6) + 2 * c * v.abs()).all()), float(off.max())
        assert float(q.double().abs().amax()) == M   # the largest is the largest code


@pytest.mark.parametrize("dtype", DTYPES)
def test_8_bits_special_rows(cuda, dtype):
    x = make(6, 200, dtype, 7)
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126
    x[3] = tiny * torch.sign(x[3].float()).to(dtype)   # the smallest numbers: squares vanish, eps decides
    for quant in ("fp8", "int8"):
        q, scale = sp.rms_norm(x, quant=quant)
        assert float(scale[0]) == 0.0 and not q[0].double().abs().any()
        assert torch.isnan(scale[1:3]).all()
        y, _ = reference(x, None, 1e-6)
        for i in (3, 4, 5):
            got = dequantised(q[i:i + 1], scale[i:i + 1])
            # no further off than a sixteenth of the row's largest (e4m3) and a subnormal scale's rounding
            assert float((got - y[i:i + 1]).abs().max()) <= float(y[i].abs().max()) / 16 + 448 * 2.0 ** -149
    y = sp.rms_norm(x)
    assert torch.isnan(y[1:3]).any(dim=1).all() and torch.isfinite(y[3:]).all() and not y[0].any()


def backward_reference(dy, h, w, dh, eps):
    """(dx, bound of dx in units of E, dw, the same of dw) in 64 bits"""
    D = h.shape[-1]
    dy, h = dy.double(), h.double()
    w = torch.ones(D, dtype=torch.float64, device=h.device) if w is None else w.double()
    _, s = reference(h, None, eps)
    n, u = h * s, dy * w
    m = (u * n).sum(-1, keepdim=True) / D
    dx = s * (u - n * m)
    size = s * (u.abs() + n.abs() * (u * n).abs().sum(-1, keepdim=True) / D)
    if dh is not None:
        dx = dx + dh.double()
        size = size + dh.double().abs()
    return dx, size, (dy * n).sum(0), (dy * n).abs().sum(0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", SIZES + [(5000, 96), (3001, 769), (2500, 2048)])
def test_backward(cuda, rows, D, dtype):
    print(f"rms_norm_backward {rows}x{D} {dtype}", flush=True)
    h, dy, dh, w = make(rows, D, dtype, 8, 2.0), make(rows, D, dtype, 9), make(rows, D, dtype, 10), weight_of(D, dtype, 11)
    c = 3 * c_of(D) + 16
    for weight, extra in ((w, None), (w.float(), dh), (None, dh)):
        dx, dw = sp.rms_norm_backward(dy, h, weight, eps=1e-5, dh=extra)
        want, size, want_w, size_w = backward_reference(dy, h, weight, extra, 1e-5)
        check("dx", dx, want, c * E * size + U[dtype] * want.abs() + TINY[dtype])
        if weight is None:
            assert dw is None
            continue
        # a thread adds its rows one after another, then the partial sums: at most rows additions
        check("dw", dw, want_w, (c + rows + 64) * E * size_w + U[weight.dtype] * want_w.abs() + TINY[weight.dtype])
    assert sp.rms_norm_backward(dy, h, w, need_dw=False)[1] is None


def test_gradient_is_the_difference_of_the_loss(cuda):
    """float32 gradients against central differences of the formula in 64 bits along random directions"""
    rows, D, eps = 7, 193, 1e-4
    x, r, w = make(rows, D, torch.float32, 12), make(rows, D, torch.float32, 13), weight_of(D, torch.float32, 14)
    a, b = make(rows, D, torch.float32, 15).double(), make(rows, D, torch.float32, 16).double()
    X, R, W = (t.clone().requires_grad_() for t in (x, r, w))
    y, h = sp.rms_norm(X, W, residual=R, eps=eps)
    ((y * a.float()).sum() + (h * b.float()).sum()).backward()
    assert torch.equal(X.grad, R.grad)

    def loss(h, w):
        return float((reference(h, w, eps)[0] * a).sum() + (h * b).sum())

    h0, w0 = (x + r).double(), w.double()
    for seed in range(3):
        d, e = make(rows, D, torch.float32, 20 + seed).double(), make(1, D, torch.float32, 30 + seed)[0].double()
        t = 1e-5
        along_h = (loss(h0 + t * d, w0) - loss(h0 - t * d, w0)) / (2 * t)
        along_w = (loss(h0, w0 + t * e) - loss(h0, w0 - t * e)) / (2 * t)
        # the difference's own error: t^2 times third derivatives (order 1) and 2^-52 of the loss over t
        own = 1e-7 * rows * D
        _, size, _, size_w = backward_reference(a.float(), h0.float(), w, b.float(), eps)
        c = 3 * c_of(D) + 16
        assert abs(float((X.grad.double() * d).sum()) - along_h) <= own + (c + 1) * E * float((size * d.abs()).sum())
        assert abs(float((W.grad.double() * e).sum()) - along_w) <= own + (c + rows + 64) * E * float((size_w * e.abs()).sum())


def test_autograd_forms(cuda):
    x, w = make(5, 40, torch.bfloat16, 17), weight_of(40, torch.bfloat16, 18)
    X, W = x.clone().requires_grad_(), w.clone().requires_grad_()
    dy = make(5, 40, torch.bfloat16, 19)
    sp.rms_norm(X, W).backward(dy)
    dx, dw = sp.rms_norm_backward(dy, x, w)
    assert torch.equal(X.grad, dx) and torch.equal(W.grad, dw)
    # only the stream goes on
    X, R, W = x.clone().requires_grad_(), x.clone().requires_grad_(), w.clone().requires_grad_()
    y, h = sp.rms_norm(X, W, residual=R)
    h.backward(dy)
    assert torch.equal(X.grad, dy) and torch.equal(R.grad, dy) and not W.grad.any()
    with torch.no_grad():
        assert not sp.rms_norm(X, W).requires_grad


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_axes(cuda, dtype):
    wide = make(30, 3 * 65, dtype, 21)
    w = weight_of(65, dtype, 22)
    x = wide[:, 65:130]                              # rows apart, an odd start
    assert torch.equal(sp.rms_norm(x, w), sp.rms_norm(x.contiguous(), w))
    t = make(65, 30, dtype, 23).T                    # neighbouring elements apart
    assert torch.equal(sp.rms_norm(t, w), sp.rms_norm(t.contiguous(), w))
    c = wide.view(5, 6, 195)[:, :, :65]
    y, h = sp.rms_norm(c, w, residual=c)
    assert y.shape == c.shape and torch.equal(y.view(30, 65), sp.rms_norm(wide[:, :65], w, residual=wide[:, :65])[0])
    one = make(1, 65, dtype, 24).expand(4, 65)       # every row the same memory
    assert torch.equal(sp.rms_norm(one, w), sp.rms_norm(one.contiguous(), w))
    assert sp.rms_norm(x[0], w).shape == (65,)
    q, scale = sp.rms_norm(c, w, quant="int8")
    assert q.shape == c.shape and scale.shape == c.shape[:-1]
    dx, dw = sp.rms_norm_backward(x, wide[:, :65], w, dh=wide[:, 130:])
    dx2, dw2 = sp.rms_norm_backward(x.contiguous(), wide[:, :65].contiguous(), w, dh=wide[:, 130:].contiguous())
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


def test_no_rows(cuda):
    x, w = torch.empty(0, 12, device=cuda), torch.ones(12, device=cuda)
    y, h = sp.rms_norm(x, w, residual=x)
    assert y.shape == (0, 12) and h.shape == (0, 12)
    dx, dw = sp.rms_norm_backward(x, x, w)
    assert dx.shape == (0, 12) and torch.equal(dw, torch.zeros_like(w))


def test_refusals(cuda):
    x, w = make(4, 8, torch.bfloat16, 1), weight_of(8, torch.bfloat16, 2)
    for bad in (lambda: sp.rms_norm(x, w[:7]), lambda: sp.rms_norm(x, w, residual=x[:3]), lambda: sp.rms_norm(x, quant="fp4"),
                lambda: sp.rms_norm(torch.ones((), device=cuda)), lambda: sp.rms_norm(x[:, :0]),
                lambda: sp.rms_norm_backward(x[:3], x, w), lambda: sp.rms_norm(x, w.cpu()[:8].repeat(2).cuda())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: sp.rms_norm(x, w.half()), lambda: sp.rms_norm(x, w, residual=x.float()),
                lambda: sp.rms_norm(x.double()), lambda: sp.rms_norm_backward(x.float(), x, w), lambda: sp.rms_norm(x, w.cpu())):
        with pytest.raises(TypeError):
            bad()


def test_graph_and_stream(cuda):
    """captured, replayed between other work, on a stream of its own; every replay is the eager result"""
    x, r, w, dy = (make(64, 1111, torch.bfloat16, s) for s in (1, 2, 3, 4))
    w = w[0].contiguous()

    def step():
        y, h = sp.rms_norm(x, w, residual=r)
        q, scale, _ = sp.rms_norm(x, w, residual=r, quant="fp8")
        return (y, h, q.view(torch.uint8), scale, *sp.rms_norm_backward(dy, h, w, dh=r))

    eager = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = step()
    for rep in range(3):
        for o in out:
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b), rep
        again = step()
        assert all(torch.equal(a, b) for a, b in zip(again, eager))
    assert math.isfinite(float(eager[0].float().sum()))
