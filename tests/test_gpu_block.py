"""block_norm, its backward pass and dropout against plain forms in 64 bits. Bounds: half a step of the type for each rounding
to it, and 2^-18 of what is added up for fp32's sums (at most 16 elements in a row and a tree of 20 levels: below 40 steps
of 2^-24, times what the reciprocal roots, the exponential and the products add)."""
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import spanqr_amd as sp

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}   # half a step of the subnormals
SUM = 2.0 ** -18


def philox(c, k):
    """Philox-4x32-10 of counters [4] of uint64 arrays below 2^32 and a key of two numbers"""
    low = np.uint64(0xFFFFFFFF)
    c, k = list(c), [np.uint64(v) for v in k]
    with np.errstate(over="ignore"):   # (modulo 2^64)
        for _ in range(10):
            a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(b >> np.uint64(32)) ^ c[1] ^ k[0], b & low, (a >> np.uint64(32)) ^ c[3] ^ k[1], a & low]
            k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return c


def numbers(rows, D, seed, index, row0=0):
    """[rows, D]: the elements' 16-bit numbers"""
    seed &= (1 << 64) - 1
    pieces = -(-D // 8)
    row = np.arange(row0, row0 + rows, dtype=np.uint64)[:, None] + np.zeros((1, pieces), np.uint64)
    c = [np.arange(pieces, dtype=np.uint64)[None, :] + 0 * row, row & np.uint64(0xFFFFFFFF), row >> np.uint64(32),
         np.full_like(row, index)]
    words = np.stack(philox(c, (seed & 0xFFFFFFFF, seed >> 32)), 2)
    return np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 3).reshape(rows, -1)[:, :D].astype(np.int64)


def kept(rows, D, p, seed, index, device="cuda"):
    return torch.from_numpy(numbers(rows, D, seed, index) >= round(65536 * p)).to(device)


def test_generator_known_answers():
    """the method's published test vectors"""
    one = np.ones(1, np.uint64)
    got = philox([0 * one] * 4, (0, 0))
    assert [int(v[0]) for v in got] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    got = philox([0xFFFFFFFF * one] * 4, (0xFFFFFFFF, 0xFFFFFFFF))
    assert [int(v[0]) for v in got] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D", [(1, 1), (5, 3), (1300, 7), (3, 8), (1, 8192), (17, 769), (2049, 24), (3, 40000), (40, 8200)])
def test_dropout(cuda, dtype, rows, D):
    x = (1.0 + torch.rand(rows, D, device=cuda)).to(dtype)
    for p, seed, index in ((0.3, 1234567890123456789, 0), (0.5, -5, 2 ** 32 - 1), (0.0, 1, 0), (1e-5, 3, 7), (65535 / 65536, 0, 1)):
        y = sp.dropout(x, p, seed, index)
        keep = kept(rows, D, p, seed, index)
        factor = 65536 / (65536 - round(65536 * p))
        want = torch.where(keep, x.double() * factor, 0.0)
        assert torch.equal(y == 0, ~keep), (p, seed)
        fits = want.abs() <= torch.finfo(dtype).max
        # the factor in fp32, the product, and its rounding to the type
        assert ((y.double() - want).abs()[fits] <= ((HALF[dtype] + 2.0 ** -23) * want.abs())[fits]).all()
        on_device = torch.tensor([seed], dtype=torch.int64, device=cuda)
        assert torch.equal(sp.dropout(x, p, on_device, index), y)


def test_dropout_forms(cuda):
    """strides, more axes, no axes, no elements, infinities, and the gradient"""
    x = torch.randn(6, 50, 33, device=cuda)
    want = sp.dropout(x, 0.4, 9, 2)
    assert torch.equal(want.view(300, 33) == 0, ~kept(300, 33, 0.4, 9, 2))
    assert torch.equal(sp.dropout(x.transpose(0, 1).contiguous().transpose(0, 1), 0.4, 9, 2), want)
    wide = torch.randn(300, 70, device=cuda)
    wide[:, 3:36] = x.view(300, 33)
    assert torch.equal(sp.dropout(wide[:, 3:36], 0.4, 9, 2), want.view(300, 33))
    assert torch.equal(sp.dropout(x[0, :1].expand(50, 33), 0.4, 9, 2) == 0, ~kept(50, 33, 0.4, 9, 2))
    assert sp.dropout(torch.ones((), device=cuda), 0.0).item() == 1.0
    assert sp.dropout(torch.ones(0, 5, device=cuda), 0.5, 1).shape == (0, 5)
    assert sp.dropout(torch.ones(5, 0, device=cuda), 0.5, 1).shape == (5, 0)
    for bad in (float("inf"), float("nan")):
        y = sp.dropout(torch.full((40, 40), bad, device=cuda), 0.5, 1)
        keep = kept(40, 40, 0.5, 1, 0)
        assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    a = torch.randn(20, 31, device=cuda, requires_grad=True)
    y = sp.dropout(a, 0.25, torch.tensor([77], device=cuda), 5)
    dy = torch.randn_like(y)
    g, = torch.autograd.grad(y, a, dy, create_graph=True)
    assert torch.equal(g, sp.dropout(dy, 0.25, 77, 5))
    # linear: the gradient of y^2's gradient is 2 factor^2
    z = sp.dropout(a, 0.25, 77, 5)
    g, = torch.autograd.grad(z.square().sum(), a, create_graph=True)
    gg, = torch.autograd.grad(g.sum(), a)
    f = kept(20, 31, 0.25, 77, 5) / 0.75
    assert torch.allclose(gg, (2 * f * f).float(), rtol=1e-6)


def test_dropout_rows_beyond_32_bits_of_elements(cuda):
    """the last rows of more than 2^32 elements"""
    rows, D = 2 ** 20 + 3, 4096
    x = torch.ones(1, D, dtype=torch.bfloat16, device=cuda).expand(rows, D)   # (copied: rows overlap)
    y = sp.dropout(x, 0.5, 11)
    want = torch.from_numpy(numbers(3, D, 11, 0, row0=2 ** 20) >= 32768).to(cuda)
    assert torch.equal(y[2 ** 20:] != 0, want)


def act(gate, kind):
    g = gate.double()
    s = torch.sigmoid(g)
    if kind is None:
        return g, torch.ones_like(g)
    return (s, s * (1 - s)) if kind == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def plain(x, r, w1, w2, gate, kind, scale, keep, factor, eps, h=None, dy=None, dh=None):
    """in 64 bits: h before its rounding and what of it is added up, then from h as it is given y, and the gradients, each with
    what is added up for it"""
    X, D = x.double(), x.shape[-1]
    W1, W2 = (torch.ones(D, device=x.device, dtype=torch.float64) if w is None else w.double() for w in (w1, w2))
    s1 = ((X * X).mean(-1, keepdim=True) + eps).rsqrt()
    n1 = X * s1
    a, slope = (torch.ones_like(X), None) if gate is None else act(gate, kind)
    k = keep * factor
    t = n1 * W1 * a * k
    out = {"h": (r.double() + scale * t, r.double().abs() + abs(scale) * t.abs())}
    if h is None:
        return out
    H = h.double()
    s2 = ((H * H).mean(-1, keepdim=True) + eps).rsqrt()
    n2 = H * s2
    out["y"] = n2 * W2, (n2 * W2).abs()
    if dy is None and dh is None:
        return out
    DY = torch.zeros_like(X) if dy is None else dy.double()
    DH = torch.zeros_like(X) if dh is None else dh.double()
    u = DY * W2
    dr = s2 * (u - n2 * (u * n2).mean(-1, keepdim=True)) + DH
    dr_sum = s2 * (u.abs() + n2.abs() * (u * n2).abs().mean(-1, keepdim=True)) + DH.abs()
    out["residual"] = dr, dr_sum
    v, v_sum = dr * k, dr_sum * k
    q, q_sum = v * W1 * a, v_sum * (W1 * a).abs()
    m, m_sum = (q * n1).mean(-1, keepdim=True), (q_sum * n1.abs()).mean(-1, keepdim=True)
    out["x"] = scale * s1 * (q - n1 * m), abs(scale) * s1 * (q_sum + n1.abs() * m_sum)
    if gate is not None:
        # (a bit more for the slope's own difference, 1 + g (1 - s))
        out["gate"] = scale * v * n1 * W1 * slope, 2 * abs(scale) * v_sum * (n1 * W1).abs() * (slope.abs() + 1)
    flat = list(range(x.dim() - 1))
    if w1 is not None:
        out["post_weight"] = (scale * v * a * n1).sum(flat), (abs(scale) * v_sum * (a * n1).abs()).sum(flat)
    if w2 is not None:
        out["weight"] = (DY * n2).sum(flat), (DY * n2).abs().sum(flat)
    out["scale"] = (q * n1).sum(), (q_sum * n1.abs()).sum()
    return out


def near(got, want, what):
    want, added = want
    assert got.shape == want.shape, what
    err, bound = (got.double() - want).abs(), HALF[got.dtype] * want.abs() + SUM * added + TINY[got.dtype]
    assert (err <= bound).all(), f"{what}: {float((err / bound.clamp_min(1e-300)).max())} times the bound"


def inputs(rows, D, dtype, wtype, gate, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    x, r, dy, dh, z = (normal(rows, D).to(dtype) for _ in range(5))
    w1, w2 = ((1 + 0.2 * normal(D)).to(wtype) for _ in range(2))
    return x, r, dy, dh, (z if gate else None), w1, w2


SIZES = [(1, 1), (3, 5), (40, 7), (5, 8), (33, 120), (70, 129), (100, 512), (65, 513), (9, 769), (1200, 2048), (600, 4100),
         (5, 8192), (3, 8200), (2, 16384), (300, 17408), (2, 20001)]


@pytest.mark.parametrize("dtype,wtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                         (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,D", SIZES)
def test_block_norm(cuda, rows, D, dtype, wtype):
    for gate, kind, p, scale in ((True, "silu", 0.1, 0.5), (False, "silu", 0.0, 1.0), (True, "sigmoid", 0.25, -1.5)):
        x, r, dy, dh, z, w1, w2 = inputs(rows, D, dtype, wtype, gate)
        how = dict(gate=z, gate_act=kind, p=p, seed=42, index=7, eps=1e-5)
        y, h = sp.block_norm(x, r, w1, w2, scale=scale, **how)
        keep, factor = kept(rows, D, p, 42, 7), 65536 / (65536 - round(65536 * p))
        want = plain(x, r, w1, w2, z, kind, scale, keep, factor, 1e-5, h, dy, dh)
        near(h, want["h"], "h")
        near(y, want["y"], "y")
        at = torch.tensor([scale], device=cuda)
        g = sp.block_norm_backward(dy, dh, x, h, w1, w2, scale=at, **how)
        for name in ("x", "residual", "gate", "post_weight", "weight", "scale"):
            if name == "gate" and z is None:
                assert g.gate is None
            else:
                near(getattr(g, name), want[name], name)
        again = sp.block_norm_backward(dy, dh, x, h, w1, w2, scale=at, **how)
        assert all(a is b or torch.equal(a, b) for a, b in zip(g, again))
        ya, ha = sp.block_norm(x, r, w1, w2, scale=at, **how)
        assert torch.equal(ya, y) and torch.equal(ha, h)


@pytest.mark.parametrize("D", [6, 96, 400, 1111, 9000])
def test_parts_left_out(cuda, D):
    """no weights, the gate as it is, one of dy and dh alone, no sums wanted, strided inputs"""
    rows = 37
    x, r, dy, dh, z, w1, w2 = inputs(rows, D, torch.bfloat16, torch.bfloat16, True, 1)
    big = torch.randn(rows, 5, D + 3, device=cuda).bfloat16()
    for i, t in enumerate((x, r, dy, dh, z)):
        big[:, i, 1:D + 1] = t
    strided = [big[:, i, 1:D + 1] for i in range(5)]
    keep = torch.ones(rows, D, device=cuda)
    y, h = sp.block_norm(x, r, gate=z, gate_act=None)
    ys, hs = sp.block_norm(strided[0], strided[1], gate=strided[4], gate_act=None)
    assert torch.equal(y, ys) and torch.equal(h, hs)
    for a, b, sa, sb in ((dy, None, strided[2], None), (None, dh, None, strided[3]), (None, None, None, None)):
        want = plain(x, r, None, None, z, None, 1.0, keep, 1.0, 1e-6, h, dy=torch.zeros_like(x) if a is None else a, dh=b)
        g = sp.block_norm_backward(a, b, x, h, gate=z, gate_act=None)
        gs = sp.block_norm_backward(sa, sb, strided[0], h, gate=strided[4], gate_act=None)
        assert g.post_weight is None and g.weight is None and g.scale is None
        for name in ("x", "residual", "gate"):
            near(getattr(g, name), want[name], name)
            assert torch.equal(getattr(g, name), getattr(gs, name))
    g = sp.block_norm_backward(dy, dh, x, h, w1, w2, need_weights=False, need_scale=True)
    assert g.post_weight is None and g.weight is None and g.scale is not None
    want = plain(x, r, w1, w2, None, None, 1.0, keep, 1.0, 1e-6, h, dy, dh)
    near(g.scale, want["scale"], "scale")
    one = sp.block_norm_backward(dy, dh, x, h, None, w2)
    assert one.post_weight is None and one.weight is not None


def test_edges(cuda):
    # rows of zeros, infinities and NaN stay in their rows; dropped infinities leave the stream as it was
    x, r, dy, dh, z, w1, w2 = inputs(6, 300, torch.float32, torch.float32, True, 2)
    x[1] = 0.0
    r[1] = 0.0
    x[3, 5] = float("nan")
    z[4, 7] = float("inf")
    y, h = sp.block_norm(x, r, w1, w2, gate=z)
    assert (y[1] == 0).all() and (h[1] == 0).all()
    assert torch.isnan(y[3]).all() and torch.isnan(h[3]).all()
    for i in (0, 1, 2, 5):
        assert torch.isfinite(y[i]).all() and torch.isfinite(h[i]).all()
    g = sp.block_norm_backward(dy, dh, x, h, w1, w2, gate=z)
    for i in (0, 1, 2, 5):
        assert all(torch.isfinite(t[i]).all() for t in (g.x, g.residual, g.gate))
    seed = 5
    keep = kept(6, 300, 0.5, seed, 0)
    z = torch.where(keep, z.nan_to_num(posinf=1.0), torch.full_like(z, float("inf")))
    x = x.nan_to_num()
    y, h = sp.block_norm(x, r, w1, w2, gate=z, gate_act=None, p=0.5, seed=seed)
    assert torch.isfinite(h).all() and torch.equal(h[~keep], r[~keep])
    # no rows: the weights' gradients are zeros
    e = torch.empty(0, 300, device=cuda)
    y, h = sp.block_norm(e, e, w1, w2)
    assert y.shape == h.shape == (0, 300)
    g = sp.block_norm_backward(e, e, e, e, w1, w2, need_scale=True)
    assert not g.weight.any() and not g.post_weight.any() and g.scale == 0 and g.x.shape == (0, 300)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gates(cuda, dtype):
    """the gate's activations and slopes over their whole range, ends and NaN included"""
    g = torch.cat([torch.linspace(-100, 100, 4001), torch.linspace(-8, 8, 4001),
                   torch.tensor([0.0, -0.0, 1e-6, -1e-6, 6e4, -6e4, float("inf"), -float("inf"), float("nan")])]).to(dtype).cuda()[:, None]
    x, r = torch.ones_like(g), torch.zeros_like(g)
    dh = torch.ones_like(g)
    for kind in ("sigmoid", "silu", None):
        want, slope = act(g, kind)
        y, h = sp.block_norm(x, r, gate=g, gate_act=kind, eps=0.0)
        d = sp.block_norm_backward(None, dh, x, h, gate=g, gate_act=kind, eps=0.0).gate
        # exp(-g)'s share: 2^-20 of it (less in fp32); s below 2^-126 may be 0, which times |g| < 2^7 is 2^-119. The slope has
        # 1 - s, off by half a step of s, 2^-24, in s (1 - s) and, times g, in s (1 + g (1 - s)): a step of s and a rounding each
        far = (g.double().abs().nan_to_num(posinf=0.0) + 1) * torch.sigmoid(g.double()) * 2.0 ** -23
        for got, w, size, more in ((h, want, want.abs(), 0.0), (d, slope, slope.abs() + torch.sigmoid(g.double()), far)):
            bound = (HALF[dtype] + 2.0 ** (-22 if dtype == torch.float32 else -19)) * size + max(TINY[dtype], 2.0 ** -119) + more
            if kind == "silu":
                w = torch.where(g.double() == -math.inf, got.double(), w)   # (-inf times 0)
            same = (got.double() == w) | ((got.double() - w).abs() <= bound) | (torch.isnan(got) & torch.isnan(w))
            assert same.all(), (kind, g[~same][:3], got[~same][:3], w[~same][:3])


def test_autograd(cuda):
    """against differences, in every input; once"""
    torch.manual_seed(3)
    x, r, dy, dh, z, w1, w2 = (None if t is None else t.requires_grad_() for t in
                               inputs(4, 24, torch.float32, torch.float32, True, 3))
    a = torch.tensor([[0.7]], device=cuda, requires_grad=True)
    leaves = (x, r, w1, w2, z, a)
    how = dict(p=0.25, seed=torch.tensor(123456789, device=cuda), index=4)

    def loss(x, r, w1, w2, z, a, f=sp.block_norm):
        y, h = f(x, r, w1, w2, gate=z, scale=a, **how)
        return (y * dy.detach()).sum() + (h * dh.detach()).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    keep, factor = kept(4, 24, 0.25, 123456789, 4), 1 / 0.75

    def in_64_bits(x, r, w1, w2, z, a):
        t = x * ((x * x).mean(-1, keepdim=True) + 1e-6).rsqrt() * w1 * (z * torch.sigmoid(z)) * keep * factor
        h = r + a * t
        y = h * ((h * h).mean(-1, keepdim=True) + 1e-6).rsqrt() * w2
        return (y * dy.detach().double()).sum() + (h * dh.detach().double()).sum()

    values = [t.detach().double() for t in leaves]
    for i, (t, g) in enumerate(zip(values, grads)):
        assert g.shape == t.shape
        for _ in range(3):
            d = torch.randn_like(t)
            step = 1e-5
            up, down = (in_64_bits(*(v + s * step * d if j == i else v for j, v in enumerate(values))) for s in (1, -1))
            slope = float((up - down) / (2 * step))
            # 2^-18 of each of the (at most 96) elements' parts, and the difference's own error of step^2
            assert abs(float((g.double() * d).sum()) - slope) <= 1e-4 * float((g.double() * d).abs().sum()) + 1e-6
    g, = torch.autograd.grad(loss(*leaves), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        g.square().sum().backward()
    # one output alone, and inputs that need no gradient
    y, h = sp.block_norm(x, r.detach(), w1, w2, gate=z.detach(), **how)
    gx, = torch.autograd.grad(h.sum(), x, retain_graph=True)
    assert gx.abs().sum() > 0
    gx, gw = torch.autograd.grad(y.sum(), (x, w2))
    assert gw.shape == w2.shape


def test_tangents_are_refused(cuda):
    x, r, dy, dh, z, w1, w2 = inputs(4, 24, torch.float32, torch.float32, True, 3)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x.clone(), torch.ones_like(x))
        for f in (lambda: sp.dropout(d, 0.5, 1), lambda: sp.block_norm(d, r), lambda: sp.block_norm(x, d),
                  lambda: sp.block_norm(x, r, gate=d), lambda: sp.block_norm_backward(d, None, x, r),
                  lambda: sp.block_norm_backward(None, d, x, r)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()


def test_refusals(cuda):
    x = torch.zeros(4, 8, device=cuda)
    h = x.half()
    w = torch.ones(8, device=cuda)
    for f in (lambda: sp.dropout(x, 1.0, 1), lambda: sp.dropout(x, -0.1, 1), lambda: sp.dropout(x, float("nan"), 1),
              lambda: sp.dropout(x, 0.5), lambda: sp.dropout(x, 0.5, 1, -1), lambda: sp.dropout(x, 0.5, 1, 1 << 32),
              lambda: sp.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64)), lambda: sp.block_norm(x, x[:2]),
              lambda: sp.block_norm(x, x, w[:3]), lambda: sp.block_norm(x, x, gate=x[:, :4]),
              lambda: sp.block_norm(x, x, gate=x, gate_act="gelu"), lambda: sp.block_norm(x, x, p=0.5),
              lambda: sp.block_norm(x, x, scale=torch.ones(2, device=cuda)),
              lambda: sp.block_norm(x[:, :0], x[:, :0]), lambda: sp.block_norm_backward(x[:1], None, x, x),
              lambda: sp.block_norm_backward(None, x[:1], x, x), lambda: sp.block_norm_backward(None, None, x, x[:1])):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: sp.dropout(x.double(), 0.5, 1), lambda: sp.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64, device=cuda)),
              lambda: sp.dropout(x, 0.5, torch.zeros(1, device=cuda)), lambda: sp.block_norm(x, h), lambda: sp.block_norm(x, x, w.half()),
              lambda: sp.block_norm(h, h, w, w.half()), lambda: sp.block_norm(x, x, scale=w[:1].double()),
              lambda: sp.block_norm(x, x, scale=torch.ones(1)), lambda: sp.block_norm(x, x, gate=h)):
        with pytest.raises(TypeError):
            f()


def test_graph_and_streams(cuda):
    """captured, with the seed and the scale changed between replays, and the eager call between them; another stream"""
    x, r, dy, dh, z, w1, w2 = inputs(130, 1000, torch.bfloat16, torch.bfloat16, True, 6)
    seed, a = torch.tensor([1], device=cuda), torch.tensor(0.5, device=cuda)

    def step():
        y, h = sp.block_norm(x, r, w1, w2, gate=z, scale=a, p=0.1, seed=seed, index=2)
        return (y, h, sp.dropout(x, 0.2, seed, 3), *sp.block_norm_backward(dy, dh, x, h, w1, w2, gate=z, scale=a, p=0.1, seed=seed,
                                                                          index=2))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        seed.fill_(i + 1)
        a.fill_(0.5 + i)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, eager))
        if i == 0:
            assert all(torch.equal(u, v) for u, v in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_slope_of_large_gates(cuda, dtype):
    """the slopes where sigmoid is next to 1, to the type's rounding and, of themselves, exp(-g)'s: -g log2 e is rounded to half a step of
    up to 128, 2^-18, which times ln 2 and with the other roundings stays below 2^-17 (bf16); in fp32 and fp16, which take
    that out, below 2^-20"""
    g = torch.linspace(0.0, 80.0, 8001, device=cuda).to(dtype)[:, None]
    x = torch.ones_like(g)
    y, h = sp.block_norm(x, torch.zeros_like(x), gate=g, gate_act="sigmoid", eps=0.0)
    s = torch.sigmoid(g.double())
    rest = torch.sigmoid(-g.double())
    more = 2.0 ** (-17 if dtype == torch.bfloat16 else -20)
    for kind, want in (("sigmoid", s * rest), ("silu", s * (1.0 + g.double() * rest))):
        got = sp.block_norm_backward(None, x, x, h, gate=g, gate_act=kind, eps=0.0).gate
        assert ((got.double() - want).abs() <= (HALF[dtype] + more) * want + TINY[dtype]).all(), kind


@pytest.mark.parametrize("rows,D,dtype", [(65536, 64, torch.bfloat16), (1 << 20, 40, torch.float32), (30000, 500, torch.float32),
                                          (20000, 2048, torch.float16), (4096, 9000, torch.float32), (16384, 8200, torch.bfloat16),
                                          (3, 1 << 20, torch.float32), (300, 100000, torch.bfloat16)])
def test_long_sums(cuda, rows, D, dtype):
    """many rows a workgroup, and rows of many pieces a thread. Half a step of fp32 for each addition in a row: within a row a
    thread's pieces (of 8, 8192 elements apart beyond 8192, 2 of them below), eight elements and a tree of 10 and 16 wavefronts; over
    rows those of a workgroup's thread, its 16 groups, and 64 parts at a time with a tree of 6; with 40 such steps for the rest"""
    from spanqr_amd import _lib
    x, r, dy, dh, z, w1, w2 = inputs(rows, D, dtype, torch.float32, True, 8)
    dy.abs_()   # (sums that grow with the rows)
    h = sp.block_norm(x, r, w1, w2, gate=z, scale=0.5)[1]
    at = torch.tensor([0.5], device=cuda)
    g = sp.block_norm_backward(dy, dh, x, h, w1, w2, gate=z, scale=at)
    parts = _lib.lib().spanqr_block_norm_backward_workspace(rows, D) // (4 * (2 * D + 1))
    in_row = max(2, -(-D // 8192)) + 8 + 10 + 16
    over_rows = -(-rows // parts) + 16 + -(-parts // 64) + 6
    y = sp.block_norm(x, r, w1, w2, gate=z, scale=0.5)[0]
    keep = torch.ones((), device=cuda, dtype=torch.float64)
    want = plain(x, r, w1, w2, z, "silu", 0.5, keep, 1.0, 1e-6, h, dy, dh)
    # a row's norms have in_row steps in their sums (half of that of themselves), the gradient's means again: 3 of them at most
    for name, got, steps in (("y", y, in_row), ("x", g.x, 3 * in_row), ("residual", g.residual, 3 * in_row),
                             ("post_weight", g.post_weight, 3 * in_row + over_rows), ("weight", g.weight, in_row + over_rows),
                             ("scale", g.scale, 3 * in_row + over_rows)):
        value, added = want[name]
        err, bound = (got.double() - value).abs(), HALF[got.dtype] * value.abs() + (steps + 40) * 2.0 ** -24 * added + TINY[got.dtype]
        assert (err <= bound).all(), (name, float((err / bound).max()))
