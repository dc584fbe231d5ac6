"""linear_cross_entropy where the ordinary cases do not reach: groups of columns without a finite logit, logits near the
ends of float32, tokens that are sure of their target, the log of the sum of exponentials.

The logits here are exact: a token is one number in the first place of x, a column one in the first of W, so a logit is one
product of at most 22 bits. What is left are the exponentials and their sum: the distance D of a logit from the maximum is
rounded, multiplied by a rounded constant and rounded again (3 E D of the exponential), the exponential itself within 2 E,
in a group and once more from the group to the whole; at most 80 additions stand behind each other. So a sum of
exponentials is within (3 D + 100) E of itself."""
import math

import pytest
import torch

import spanqr_amd as sp

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.bfloat16, torch.float16]
# few tokens (1 to 16, 17 to 32), and the three tiles of the others
SIZES = [(1, 8, 33), (3, 8, 500), (20, 8, 1000), (32, 72, 4000), (33, 8, 130), (70, 136, 1111), (300, 64, 5000),
         (2048, 8, 20000)]


def place(column, H):
    """[n] as [n, H] with zeros behind"""
    t = torch.zeros(column.shape[0], H, dtype=column.dtype, device=column.device)
    t[:, 0] = column
    return t


def exact(s, w, t):
    """loss, softmax and the largest distance of a logit from the maximum, in 64 bits, for z = s w^T; -inf logits allowed"""
    z = s.double()[:, None] * w.double()[None]
    z = torch.where(z.abs() >= 2.0 ** 128, torch.sign(z) * math.inf, z)   # as float32 has it
    zt = z.gather(1, t[:, None])
    m = z.amax(1, keepdim=True)
    others = z.clone().scatter_(1, t[:, None], -math.inf)
    M = torch.maximum(others.amax(1, keepdim=True), zt)
    loss = torch.where(zt == M, torch.log1p(torch.exp(others - M).sum(1, keepdim=True)),
                       M - zt + torch.log(torch.exp(z - M).sum(1, keepdim=True)))[:, 0]
    far = torch.where(z > m - 200, m - z, torch.zeros_like(z)).amax(1)   # further ones add nothing
    return loss, torch.softmax(z - m, 1), far


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", SIZES)
def test_groups_without_a_finite_logit(cuda, N, H, V, dtype):
    """columns that are out (-inf), whole groups of them, beside logits far below 0: they take no part"""
    print(f"linear_cross_entropy {N}x{H}x{V} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(31)
    w = (-100.0 + 5.0 * torch.randn(V, generator=g, device="cuda")).to(dtype)
    s = (1.0 + 1.5 * torch.rand(N, generator=g, device="cuda")).to(dtype)
    out = torch.rand(V, generator=g, device="cuda") < 0.1
    out[V // 4:V // 4 + (V + 1) // 2] = True
    t = torch.nonzero(~out)[:, 0][torch.randint(0, int((~out).sum()), (N,), generator=g, device="cuda")]
    w[out] = -math.inf
    want, p, far = exact(s, w, t)
    tol = want.abs() * E * 4 + (3 * far + 100) * E
    x, W = place(s, H), place(w, H)
    loss = sp.linear_cross_entropy(x, W, t, reduction="none")
    assert bool(((loss.double() - want).abs() <= tol).all()), float((loss.double() - want).abs().max())
    total, none, dw = sp.linear_cross_entropy_grad(x, W, t, reduction="sum", need_dx=False)
    assert bool(torch.isfinite(dw).all()) and not dw[out].any() and not dw[:, 1:].any()
    G = p.scatter_add(1, t[:, None], -torch.ones(N, 1, device=cuda, dtype=torch.float64))
    X = s.double()
    # two roundings of an element to 16 bits, float16's absolute part, the sum over the tokens, the result's own rounding
    small = 2.0 ** -24 + 2.0 ** -35 if dtype == torch.float16 else 0.0
    dG = G.abs() * (2.1 * U[dtype] + 2 * (3 * far[:, None] + 100) * E) + small * (p > 0)
    dG += 4 * (3 * far[:, None] + 100) * E * (G < 0)   # the target's: of 1, not of 1 - p
    want_w = (G * X[:, None]).sum(0)
    tol_w = (dG * X[:, None]).sum(0) + (N + 16) * E * (G.abs() * X[:, None]).sum(0) + U[dtype] * want_w.abs() * 1.01 + 2.0 ** -25
    assert bool(((dw[:, 0].double() - want_w).abs() <= tol_w).all())
    assert bool(((total.double() - want.sum()).abs() <= tol.sum() + 2 * E * want.sum()).all())


@pytest.mark.parametrize("N", [1, 20, 40, 300])
def test_logits_at_the_ends_of_float32(cuda, N):
    """bfloat16's lowest value as a mask (finite or -inf as a logit), and rows whose largest logit is near float32's ends"""
    H, V, dtype = 8, 700, torch.bfloat16
    lowest = torch.finfo(dtype).min
    g = torch.Generator(device="cuda").manual_seed(32)
    w = torch.randn(V, generator=g, device="cuda").to(dtype)
    w[100:420] = lowest
    t = torch.randint(0, 100, (N,), generator=g, device="cuda")
    for at in (1.0, 2.0):                       # the masked logits: lowest itself, -inf
        s = torch.full((N,), at, dtype=dtype, device=cuda)
        want, p, far = exact(s, w, t)
        x, W = place(s, H), place(w, H)
        loss, dx, dw = sp.linear_cross_entropy_grad(x, W, t, reduction="none")
        assert bool(((loss.double() - want).abs() <= 4 * E * want + (3 * far + 100) * E).all())
        assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(dw).all()) and not dw[100:420].any()
    s = torch.ones(N, dtype=dtype, device=cuda)
    for top in (-3.0e38, 3.0e38, -2.0e38, 2.5e38, 1e30, -1e30, 1e8, -1e8, 69632.0, -60000.0):
        w = torch.full((V,), lowest, dtype=dtype, device=cuda)
        w[::7] = top                            # 100 of one size, the others far below
        t = 7 * torch.randint(0, 100, (N,), generator=g, device="cuda")
        loss = sp.linear_cross_entropy(place(s, H), place(w, H), t, reduction="none")
        assert bool(((loss.double() - math.log(100.0)).abs() <= 200 * E).all()), (top, loss[:3])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", SIZES)
def test_small_losses(cuda, N, H, V, dtype):
    """a token that is sure of its target: what the other columns leave, from a tenth of a nat to 1e-20, as exactly as a
    large loss (relative, not beside the logits), and the gradients of such tokens"""
    print(f"linear_cross_entropy {N}x{H}x{V} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(33)
    best = int(torch.randint(0, V, (1,), generator=g, device="cuda"))
    w = (0.5 * torch.randn(V, generator=g, device="cuda")).clamp(-1.5, 1.5).to(dtype)
    w[best] = math.log(V) + 1.0
    s = (1.0 + 2.0 * torch.rand(N, generator=g, device="cuda")).to(dtype)
    s[0] = 1.0
    t = torch.full((N,), best, device=cuda)
    want, p, far = exact(s, w, t)
    assert float(want.max()) < 0.9 and float(far.max()) < 60.0
    c = (3 * far + 100) * E
    x, W = place(s, H), place(w, H)
    loss = sp.linear_cross_entropy(x, W, t, reduction="none")
    rel = (loss.double() - want).abs() / want
    assert bool((rel <= c).all()), float((rel / c).max())
    one, none, dw = sp.linear_cross_entropy_grad(x[:1], W, t[:1], reduction="sum", need_dx=False)
    assert torch.equal(one, loss[0]) or abs(float(one) - float(want[0])) <= float(c[0] * want[0])
    total, dx, dw = sp.linear_cross_entropy_grad(x, W, t, reduction="sum")
    assert abs(float(total) - float(want.sum())) <= float((c * want).sum() + 2 * E * want.sum())
    # the target's element of G is expm1(-loss): relative, too (float16 has G times 2^10 and then its smallest number)
    u, small = U[dtype], 2.0 ** -24 if dtype == torch.float16 else 0.0
    G = p.clone()
    G[:, best] = torch.expm1(-want)
    X, Y = s.double(), w.double()
    # (float16's p is relative to its group's largest, the target not among them: that is below 1 / V^0.5 here)
    dG = G.abs() * (2.1 * u + 2 * c[:, None]) + small * (G.abs().amax(1, keepdim=True) + 2.0 ** -11)
    want_x, want_w = (G * Y).sum(1), (G * X[:, None]).sum(0)
    tol_x = (dG * Y.abs()).sum(1) + (V + 16) * E * (G.abs() * Y.abs()).sum(1) + u * want_x.abs() * 1.01 + small
    tol_w = (dG * X[:, None]).sum(0) + (N + 16) * E * (G.abs() * X[:, None]).sum(0) + u * want_w.abs() * 1.01 + small
    assert bool(((dx[:, 0].double() - want_x).abs() <= tol_x).all())
    assert bool(((dw[:, 0].double() - want_w).abs() <= tol_w).all())


@pytest.mark.parametrize("N", [3, 300])
def test_small_gradients_under_a_scale(cuda, N):
    """float16, losses of 1e-9 to 1e-6 and a loss scale that takes their gradients into range: the other columns' share, which
    lies below float16's numbers next to the target's, is there"""
    H, V, dtype, scale = 8, 256, torch.float16, 2.0 ** 20
    g = torch.Generator(device="cuda").manual_seed(34)
    w = torch.randn(V, generator=g, device="cuda").to(dtype)
    w[5] = 22.0
    s = torch.linspace(0.9, 1.0, N, device=cuda).to(dtype)
    t = torch.full((N,), 5, device=cuda)
    want, p, far = exact(s, w, t)
    assert 1e-9 < float(want.min()) and float(want.max()) < 1e-6
    _, _, dw = sp.linear_cross_entropy_grad(place(s, H), place(w, H), t, reduction="sum", grad_scale=scale, need_dx=False)
    G = p.clone()
    G[:, 5] = torch.expm1(-want)
    want_w = (G * s.double()[:, None]).sum(0) * scale
    # G is held times 2^10, and a smallest number of float16 is 2^-24
    tol = (G.abs() * (2.1 * U[dtype] + 400 * E) + 2.0 ** -34).sum(0) * scale + U[dtype] * want_w.abs() * 1.01 + 2.0 ** -24
    off = (dw[:, 0].double() - want_w).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    # and no column is lost
    assert bool((dw[:, 0] != 0).all())


def test_more_tokens_than_a_launch_takes(cuda):
    """2^24 tokens and some: pieces, each of fewer than 2^32 threads"""
    N, H, V, dtype = (1 << 24) + 5, 8, 16, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(35)
    s = (torch.rand(N, generator=g, device="cuda") + 1.0).to(dtype)
    w = torch.randn(V, generator=g, device="cuda").to(dtype)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    loss = sp.linear_cross_entropy(place(s, H), place(w, H), t, reduction="none")
    for at in range(0, N, 1 << 22):
        want, _, far = exact(s[at:at + (1 << 22)], w, t[at:at + (1 << 22)])
        assert bool(((loss[at:at + (1 << 22)].double() - want).abs() <= 4 * E * want + (3 * far + 100) * E).all()), at


def abi_call(x, W, t, reduction, ws, grads, lse=None):
    """the C entry point with a workspace that is given"""
    from spanqr_amd import _lib
    N, H, V = x.shape[0], x.shape[1], W.shape[0]
    loss = torch.full((N if reduction == _lib.REDUCE_NONE else 1,), 7.0, device=x.device)
    dx, dw = (torch.empty_like(v) if grads & bit else None for v, bit in ((x, 1), (W, 2)))
    ptr = lambda v: None if v is None else v.data_ptr()   # noqa: E731
    rc = _lib.lib().spanqr_linear_cross_entropy(
        _lib.BF16 if x.dtype == torch.bfloat16 else _lib.FP16, reduction, N, H, V, x.data_ptr(), x.stride(0), W.data_ptr(),
        W.stride(0), t.data_ptr(), -100, None, None, loss.data_ptr(), ptr(lse), ptr(dx), ptr(dw), ws.data_ptr(), ws.numel(),
        torch.cuda.current_stream().cuda_stream)
    _lib.check(rc)
    return loss, dx, dw


@pytest.mark.parametrize("grads", [1, 3])
@pytest.mark.parametrize("N,H,V", [(1000, 136, 5000), (300, 768, 1024), (64, 64, 3000)])
def test_a_workspace_for_more_tokens(cuda, N, H, V, grads):
    """what the query gives for N tokens, and the least that it gives, hold fewer tokens; the bytes behind the workspace stay,
    and dx's parts, which adapt to it, change no more than their sums' order"""
    from spanqr_amd import _lib
    g = torch.Generator(device="cuda").manual_seed(36)
    x = torch.randn(N, H, generator=g, device="cuda").bfloat16()
    W = (torch.randn(V, H, generator=g, device="cuda") * (2.5 / math.sqrt(H))).bfloat16()
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    for most in (0, 16 << 20, 1 << 32):
        nbytes = _lib.lib().spanqr_linear_cross_entropy_workspace(_lib.BF16, N, H, V, grads, most)
        room = torch.full((nbytes + 4096,), 77, dtype=torch.uint8, device=cuda)
        for n in sorted({1, 2, 17, 32, 33, 64, 65, 255, 256, 257, N - 1, N}):
            if n > N:
                continue
            print(f"linear_cross_entropy {n} of {N}x{H}x{V}, {nbytes} bytes", flush=True)
            loss, dx, dw = abi_call(x[:n], W, t[:n], _lib.REDUCE_SUM, room[:nbytes], grads)
            assert bool((room[nbytes:] == 77).all())
            want = sp.linear_cross_entropy_grad(x[:n], W, t[:n], reduction="sum")
            for a, b in ((loss[0], want[0]), (dx, want[1]), (dw, want[2])):
                if a is not None:
                    a, b = a.double(), b.double()
                    # (one rounding to bfloat16 of sums that differ in their order)
                    assert float((a - b).norm()) <= 2.0 ** -8 * float(b.norm()) + 1e-6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,V", SIZES)
def test_log_of_the_sum_of_exponentials(cuda, N, H, V, dtype):
    """the C entry point's lse: of every token, whatever its target, with and without gradients, in pieces of the tokens"""
    from spanqr_amd import _lib
    print(f"linear_cross_entropy {N}x{H}x{V} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(37)
    w = (4.0 * torch.randn(V, generator=g, device="cuda")).to(dtype)
    w[1::5] = -math.inf
    s = (0.5 + torch.rand(N, generator=g, device="cuda")).to(dtype)
    z = s.double()[:, None] * w.double()[None]
    want = torch.logsumexp(z, 1)
    far = torch.where(z > -math.inf, z.amax(1, keepdim=True) - z, torch.zeros_like(z)).amax(1)
    tol = 4 * E * want.abs() + 4 * E * z.amax(1).abs() + (3 * far + 100) * E
    x, W = place(s, H), place(w, H)
    best = z.argmax(1)
    for t in (best, torch.full_like(best, -100), torch.full_like(best, V + 3),
              torch.where(torch.arange(N, device=cuda) % 2 == 0, best, torch.full_like(best, -100)),
              torch.ones_like(best) if V > 1 else best):       # (column 1 is out)
        for grads in (0, 2):
            nbytes = _lib.lib().spanqr_linear_cross_entropy_workspace(_lib.BF16, N, H, V, grads, 0)
            lse = torch.full((N + 8,), 7.0, device=cuda)
            abi_call(x, W, t, _lib.REDUCE_MEAN, torch.empty(nbytes, dtype=torch.uint8, device=cuda), grads, lse)
            assert bool((lse[N:] == 7.0).all())
            assert bool(((lse[:N].double() - want).abs() <= tol).all()), float(((lse[:N].double() - want).abs() / tol).max())
