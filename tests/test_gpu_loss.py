"""linear_cross_entropy and linear_cross_entropy_grad against the formulas in 64 bits.

The bounds, element by element: a logit is a sum of H products that are exact in fp32, so it is within d = (H + 16) 2^-24
sum|x_k w_jk| of its value, and so are lse and the target's logit; exp and log add a few roundings. An element of
G = exp(z - lse) - [target] is held in the 16-bit type after at most two roundings (u each: 2^-8 bfloat16, 2^-11 float16;
float16 has an absolute part below 2^-14), and dx = a G W is a sum of V products with the same growth of fp32 roundings, rounded once."""
import math

import pytest
import torch

import spanqr_amd as sp

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
DTYPES = [torch.bfloat16, torch.float16]
SIZES = [(1, 1, 1), (1, 8, 2), (2, 3, 5), (3, 64, 31), (5, 63, 32), (7, 65, 33), (16, 32, 64), (17, 40, 100), (64, 128, 256),
         (65, 72, 257), (33, 200, 1000), (100, 264, 1025), (1, 1024, 4000), (4, 768, 3001), (129, 96, 511), (300, 520, 700),
         (257, 257, 257), (520, 320, 1300)]


def make(N, H, V, dtype, seed, ignored=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, H, generator=g, device="cuda").to(dtype)
    W = (torch.randn(V, H, generator=g, device="cuda") * (2.5 / math.sqrt(H))).to(dtype)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    t[torch.rand(N, generator=g, device="cuda") < ignored] = -100
    return x, W, t


def reference(x, W, t, weights=None):
    """per token loss, G (unscaled), and the bounds of both, in 64 bits"""
    x, W = x.double(), W.double()
    N, H, V = x.shape[0], x.shape[1], W.shape[0]
    z = x @ W.T
    d = ((H + 16) * E * (x.abs() @ W.abs().T)).amax(1)
    lse = torch.logsumexp(z, 1)
    kept = t != -100
    w = kept.double() if weights is None else torch.where(kept, weights.double(), torch.zeros_like(lse))
    at = torch.where(kept, t, torch.zeros_like(t))
    zt = z.gather(1, at[:, None])[:, 0]
    loss = w * (lse - zt)
    loss_tol = w.abs() * (2 * d + 8 * E * (lse.abs() + zt.abs() + z.abs().amax(1) + 4))
    p = torch.exp(z - lse[:, None])
    G = p.clone()
    G[torch.arange(N, device=x.device), at] -= 1.0
    return loss, loss_tol, G * w[:, None], d, w, p


def bounds(x, W, G, d, w, dtype):
    """of sum_j G_ij W_jh and of sum_i G_ij x_ih"""
    u = U[dtype]
    # p's absolute part (float16): below 2^-14 of a piece's largest exponential, which is at most 1 after the factor
    # (G's own: its elements are held times 2^10 and the power of 2 that takes the largest weight to [1, 2))
    small = w.abs()[:, None] * 2.0 ** -24 + w.abs().max() * 2.0 ** -35 if dtype == torch.float16 else 0.0
    # the target's element is exp(z - lse) - 1: its error is that of the logits
    dG = G.abs() * (2.1 * u + 2.1 * d[:, None] + 64 * E) + 2.1 * d[:, None] * w.abs()[:, None] * (G.abs() > 0) + small
    V, N = W.shape[0], x.shape[0]
    a = dG @ W.double().abs() + (V + 16) * E * (G.abs() @ W.double().abs())
    b = dG.T @ x.double().abs() + (N + 16) * E * (G.abs().T @ x.double().abs())
    return a, b


def check(what, got, want, bound):
    assert got.shape == want.shape, what
    d = (got.double() - want).abs()
    ok = d <= bound
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} outside, worst {float((d / bound).nan_to_num().max()):.3g}"


def check_call(x, W, t, reduction, got, weights=None, scale=1.0, dtype=None):
    dtype = dtype or x.dtype
    loss, dx, dw = got
    L, tol, G, d, w, _ = reference(x, W, t, weights)
    n = max(1, int((t != -100).sum())) if reduction == "mean" else 1
    if reduction == "none":
        check("loss", loss, L, tol)
    else:
        check("loss", loss, L.sum() / n, tol.sum() / n + 2 * E * L.sum().abs() / n)
    a, b = bounds(x, W, G, d, w, dtype)
    f = scale / n
    if dx is not None:
        want = (G @ W.double()) * f
        check("dx", dx, want, a * abs(f) + U[dtype] * want.abs() * 1.01 + TINY[dtype])
    if dw is not None:
        want = (G.T @ x.double()) * f
        check("dw", dw, want, b * abs(f) + U[dtype] * want.abs() * 1.01 + TINY[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", SIZES)
def test_loss_and_gradients(cuda, N, H, V, dtype):
    print(f"linear_cross_entropy {N}x{H}x{V} {dtype}", flush=True)
    x, W, t = make(N, H, V, dtype, 1)
    check_call(x, W, t, "none", (sp.linear_cross_entropy(x, W, t, reduction="none"), None, None))
    check_call(x, W, t, "mean", (sp.linear_cross_entropy(x, W, t.int()), None, None))
    check_call(x, W, t, "mean", sp.linear_cross_entropy_grad(x, W, t))
    got = sp.linear_cross_entropy_grad(x, W, t, reduction="sum")
    check_call(x, W, t, "sum", got)
    again = sp.linear_cross_entropy_grad(x, W, t, reduction="sum")
    assert all(torch.equal(a, b) for a, b in zip(got, again))   # the same bits
    loss, dx, none = sp.linear_cross_entropy_grad(x, W, t, reduction="sum", need_dw=False)
    assert none is None and torch.equal(dx, got[1]) and torch.equal(loss, got[0])
    loss, none, dw = sp.linear_cross_entropy_grad(x, W, t, reduction="sum", need_dx=False)
    assert none is None and torch.equal(dw, got[2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", [(2100, 136, 9001), (4111, 264, 20000), (700, 1032, 33000), (2304, 2048, 8192)])
def test_large(cuda, N, H, V, dtype):
    """the largest tiles, dx over several parts of the vocabulary, pieces of the tokens"""
    print(f"linear_cross_entropy {N}x{H}x{V} {dtype}", flush=True)
    x, W, t = make(N, H, V, dtype, 21)
    check_call(x, W, t, "none", (sp.linear_cross_entropy(x, W, t, reduction="none"), None, None))
    check_call(x, W, t, "mean", sp.linear_cross_entropy_grad(x, W, t))
    check_call(x, W, t, "mean", sp.linear_cross_entropy_grad(x, W, t, max_workspace=100 << 20))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", [(4096, 4096, 1024), (1024, 4096, 4096), (4096, 2048, 4096), (3999, 4001, 4099), (2001, 2049, 33003)])
def test_largest_tiles(cuda, N, H, V, dtype):
    """each product in 256 x 256 tiles, whole and cut ones, straight, in parts of the vocabulary and in pieces of the
    tokens; the tokens that share a target column or a row's last 64 are many enough to reach every element of a tile"""
    print(f"linear_cross_entropy {N}x{H}x{V} {dtype}", flush=True)
    x, W, t = make(N, H, V, dtype, 22, ignored=0.02)
    check_call(x, W, t, "none", (sp.linear_cross_entropy(x, W, t, reduction="none"), None, None))
    check_call(x, W, t, "mean", sp.linear_cross_entropy_grad(x, W, t))
    check_call(x, W, t, "sum", sp.linear_cross_entropy_grad(x, W, t, reduction="sum", max_workspace=N * V))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", [(1, 512, 1111), (2, 136, 40), (15, 72, 3000), (16, 640, 257), (31, 65, 500), (32, 264, 2001)])
def test_few_tokens_round_once(cuda, N, H, V, dtype):
    """up to 32 tokens p and G have a second row with what their rounding drops: what is left of an element's error is the
    square of one rounding, twice. Rounding is monotone, so a gradient lies between the rounded ends of what that allows."""
    print(f"linear_cross_entropy {N}x{H}x{V} {dtype}", flush=True)
    x, W, t = make(N, H, V, dtype, 23, ignored=0.0)
    loss, dx, dw = sp.linear_cross_entropy_grad(x, W, t, reduction="sum")
    L, tol, G, d, w, _ = reference(x, W, t)
    check("loss", loss, L.sum(), tol.sum() + 2 * E * L.sum().abs())
    u = U[dtype]
    small = 2.0 ** -24 + 2.0 ** -35 if dtype == torch.float16 else 0.0   # float16's absolute part, as in bounds()
    dG = G.abs() * (2.1 * u * u + 2.1 * d[:, None] + 64 * E) + 2.1 * d[:, None] + small
    X, Y = x.double(), W.double()
    for what, got, want, error in (("dx", dx, G @ Y, dG @ Y.abs() + (V + 16) * E * (G.abs() @ Y.abs())),
                                   ("dw", dw, G.T @ X, dG.T @ X.abs() + (N + 16) * E * (G.abs().T @ X.abs()))):
        low, high = (want - error).to(dtype), (want + error).to(dtype)
        assert bool(((got >= low) & (got <= high)).all()), what


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", [(7, 65, 33), (300, 128, 520), (64, 200, 1000)])
def test_weights_and_scale(cuda, N, H, V, dtype):
    x, W, t = make(N, H, V, dtype, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(N, generator=g, device="cuda") * torch.exp(2 * torch.randn(N, generator=g, device="cuda"))
    check_call(x, W, t, "sum", sp.linear_cross_entropy_grad(x, W, t, reduction="sum", row_weight=w), w)
    small = w.abs() * 2.0 ** -20    # as an incoming gradient of a mean: G itself stays in range
    loss, dx, dw = sp.linear_cross_entropy_grad(x.bfloat16(), W.bfloat16(), t, reduction="sum", row_weight=small)
    check_call(x.bfloat16(), W.bfloat16(), t, "sum", (loss, dx, dw), small)
    check_call(x, W, t, "mean", sp.linear_cross_entropy_grad(x, W, t, grad_scale=1024.0), scale=1024.0)
    s = torch.full((1,), 3.0, device=cuda)
    check_call(x, W, t, "none", sp.linear_cross_entropy_grad(x, W, t, reduction="none", grad_scale=s), scale=3.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces_of_the_tokens(cuda, dtype):
    """a workspace that holds 256 tokens at a time"""
    N, H, V = 900, 136, 777
    x, W, t = make(N, H, V, dtype, 4)
    whole = sp.linear_cross_entropy_grad(x, W, t)
    cut = sp.linear_cross_entropy_grad(x, W, t, max_workspace=0)
    check_call(x, W, t, "mean", whole)
    check_call(x, W, t, "mean", cut)
    per = sp.linear_cross_entropy(x, W, t, reduction="none", max_workspace=0)
    check_call(x, W, t, "none", (per, None, None))


def test_gradient_is_the_difference_of_the_loss(cuda):
    """both gradients along random directions, against central differences of the loss in 64 bits"""
    N, H, V, dtype = 24, 48, 300, torch.float16
    x, W, t = make(N, H, V, dtype, 5)
    X, P = x.clone().requires_grad_(), W.clone().requires_grad_()
    loss = sp.linear_cross_entropy(X, P, t, reduction="sum")
    loss.backward()
    _, _, G, d, w, _ = reference(x, W, t)
    a, b = bounds(x, W, G, d, w, dtype)

    def f(x, W):
        return float(reference(x, W, t)[0].sum())

    g = torch.Generator(device="cuda").manual_seed(6)
    step = 1e-5
    for _ in range(3):
        dx = torch.randn(N, H, generator=g, device="cuda", dtype=torch.float64)
        dW = torch.randn(V, H, generator=g, device="cuda", dtype=torch.float64)
        along_x = (f(x.double() + step * dx, W) - f(x.double() - step * dx, W)) / (2 * step)
        along_W = (f(x, W.double() + step * dW) - f(x, W.double() - step * dW)) / (2 * step)
        own = 1e-6 * abs(along_x) + 1e-4   # step^2 times third derivatives, 2^-52 of the loss over the step
        tol = float(((a + U[dtype] * X.grad.double().abs() + TINY[dtype]) * dx.abs()).sum()) + own
        assert abs(float((X.grad.double() * dx).sum()) - along_x) <= tol
        tol = float(((b + U[dtype] * P.grad.double().abs() + TINY[dtype]) * dW.abs()).sum()) + own
        assert abs(float((P.grad.double() * dW).sum()) - along_W) <= tol


@pytest.mark.parametrize("dtype", DTYPES)
def test_autograd_forms(cuda, dtype):
    x, W, t = make(50, 72, 130, dtype, 7)
    for reduction in ("mean", "sum"):
        X, P = x.clone().requires_grad_(), W.clone().requires_grad_()
        loss = sp.linear_cross_entropy(X, P, t, reduction=reduction)
        (loss * 8.0).backward()
        want = sp.linear_cross_entropy_grad(x, W, t, reduction=reduction, grad_scale=8.0)
        assert torch.equal(loss.detach(), want[0]) and torch.equal(X.grad, want[1]) and torch.equal(P.grad, want[2])
    X, P = x.clone().requires_grad_(), W.clone().requires_grad_()
    per = torch.linspace(0.0, 2.0, 50, device=cuda)
    sp.linear_cross_entropy(X, P, t, reduction="none").backward(per)
    want = sp.linear_cross_entropy_grad(x, W, t, reduction="sum", row_weight=per)
    assert torch.equal(X.grad, want[1]) and torch.equal(P.grad, want[2])
    X = x.clone().requires_grad_()
    sp.linear_cross_entropy(X, W, t).backward()
    assert X.grad is not None
    with torch.no_grad():
        assert not sp.linear_cross_entropy(X, W, t).requires_grad


@pytest.mark.parametrize("dtype", DTYPES)
def test_ignored_and_bad_targets(cuda, dtype):
    x, W, t = make(70, 40, 90, dtype, 8)
    none = torch.full_like(t, -100)
    loss, dx, dw = sp.linear_cross_entropy_grad(x, W, none)
    assert float(loss) == 0.0 and not dx.any() and not dw.any()
    assert not sp.linear_cross_entropy(x, W, none, reduction="none").any()
    # an index that is a column can be the one to ignore
    t = t.clamp_min(0)
    t[::7] = 5
    as_usual = torch.where(t == 5, torch.full_like(t, -100), t)
    for a, b in zip(sp.linear_cross_entropy_grad(x, W, t, ignore_index=5), sp.linear_cross_entropy_grad(x, W, as_usual)):
        assert torch.equal(a, b)
    for bad in (90, -1, 1 << 40):
        u = t.clone()
        u[3] = bad
        per = sp.linear_cross_entropy(x, W, u, reduction="none")
        assert torch.isnan(per[3]) and torch.isfinite(per[:3]).all() and torch.isfinite(per[4:]).all()
        loss, dx, dw = sp.linear_cross_entropy_grad(x, W, u)
        assert torch.isnan(loss) and torch.isnan(dx[3]).all() and torch.isfinite(dx[4:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_and_infinite_logits(cuda, dtype):
    """logits of several hundred (a sure prediction, right and wrong), columns that are out (-inf), overflow to inf"""
    N, H, V = 40, 64, 333
    x, W, t = make(N, H, V, dtype, 9, ignored=0.0)
    W = (W.float() * 20).to(dtype)
    check_call(x, W, t, "sum", sp.linear_cross_entropy_grad(x, W, t, reduction="sum"))
    best = (x.double() @ W.double().T).argmax(1)
    check_call(x, W, best, "sum", sp.linear_cross_entropy_grad(x, W, best, reduction="sum"))
    # a column whose logit is -inf takes no part; as a target its loss is inf
    x1 = x.abs() + 0.5
    W1 = W.clone()
    W1[7] = float("-inf")
    W1[100:200] = float("-inf")          # whole pieces
    keep = torch.ones(V, dtype=torch.bool, device=cuda)
    keep[7] = False
    keep[100:200] = False
    t1 = torch.where(keep[t], t, torch.zeros_like(t))
    L = torch.logsumexp((x1.double() @ W1.double()[keep].T), 1) - (x1.double() * W1.double()[t1]).sum(1)
    per = sp.linear_cross_entropy(x1, W1, t1, reduction="none")
    tol = 2 * (H + 16) * E * (x1.double().abs() @ W.double().abs().T).amax(1) + 64 * E * L.abs().clamp_min(100.0)
    check("loss", per, L, tol)
    t1[0] = 7
    assert float(sp.linear_cross_entropy(x1, W1, t1, reduction="none")[0]) == float("inf")
    x2 = x.clone()
    x2[5] = float("inf")
    per = sp.linear_cross_entropy(x2, W, t, reduction="none")
    assert torch.isnan(per[5]) and torch.isfinite(per[:5]).all() and torch.isfinite(per[6:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(cuda, dtype):
    N, H, V = 90, 65, 201
    wide, wW = make(N, 3 * H, V, dtype, 10)[:2]
    t = make(N, H, V, dtype, 11)[2]
    for x, W in ((wide[:, 1:1 + H], wW[:, 70:70 + H]), (wide[:, :H], wW[:, H:2 * H]),
                 (wide[:H].T[:N].contiguous().T.contiguous()[:, :H], wW[:, :H])):
        x = x[:N]
        tt = t[:x.shape[0]]
        a = sp.linear_cross_entropy_grad(x, W, tt)
        b = sp.linear_cross_entropy_grad(x.contiguous(), W.contiguous(), tt)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    Wt = wW[:, :H].T.contiguous().T      # columns lie together
    a = sp.linear_cross_entropy_grad(wide[:, :H], Wt, t)
    assert all(torch.equal(p, q) for p, q in zip(a, sp.linear_cross_entropy_grad(wide[:, :H], wW[:, :H], t)))
    one = wide[:1, :H].expand(N, H)      # every token the same memory
    a = sp.linear_cross_entropy_grad(one, wW[:, :H], t)
    assert all(torch.equal(p, q) for p, q in zip(a, sp.linear_cross_entropy_grad(one.contiguous(), wW[:, :H], t)))
    twice = torch.stack([t, t], 1)[:, 0]
    assert torch.equal(sp.linear_cross_entropy(one, wW[:, :H], twice), a[0])


def test_no_tokens(cuda):
    x, W = torch.empty(0, 16, dtype=torch.bfloat16, device=cuda), torch.ones(33, 16, dtype=torch.bfloat16, device=cuda)
    t = torch.empty(0, dtype=torch.int64, device=cuda)
    loss, dx, dw = sp.linear_cross_entropy_grad(x, W, t)
    assert float(loss) == 0.0 and dx.shape == (0, 16) and dw.shape == (33, 16) and not dw.any()
    assert sp.linear_cross_entropy(x, W, t, reduction="none").shape == (0,)


def test_refusals(cuda):
    x, W, t = make(4, 8, 10, torch.bfloat16, 12)
    for bad in (lambda: sp.linear_cross_entropy(x, W[:, :7], t), lambda: sp.linear_cross_entropy(x, W, t[:3]),
                lambda: sp.linear_cross_entropy(x[0], W, t), lambda: sp.linear_cross_entropy(x, W, t, reduction="max"),
                lambda: sp.linear_cross_entropy_grad(x, W, t, row_weight=torch.ones(3, device=cuda)),
                lambda: sp.linear_cross_entropy(x, W[:0], t),
                lambda: sp.linear_cross_entropy_grad(x, W, t, grad_scale=torch.ones(2, device=cuda))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: sp.linear_cross_entropy(x.float(), W.float(), t), lambda: sp.linear_cross_entropy(x, W.half(), t),
                lambda: sp.linear_cross_entropy(x, W, t.float()),
                lambda: sp.linear_cross_entropy_grad(x, W, t, row_weight=torch.ones(4, device=cuda).double())):
        with pytest.raises(TypeError):
            bad()


def test_graph_and_streams(cuda):
    """captured and replayed between eager calls; two streams at once"""
    x, W, t = make(130, 200, 555, torch.bfloat16, 13)
    eager = sp.linear_cross_entropy_grad(x, W, t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sp.linear_cross_entropy_grad(x, W, t)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = sp.linear_cross_entropy_grad(x, W, t)
    for rep in range(3):
        for o in out:
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), rep
        assert all(torch.equal(a, b) for a, b in zip(sp.linear_cross_entropy_grad(x, W, t), eager))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append([sp.linear_cross_entropy_grad(x, W, t) for _ in range(3)])
    torch.cuda.synchronize()
    for runs in got:
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(r, eager))
