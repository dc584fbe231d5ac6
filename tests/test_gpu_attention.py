"""attention and its backward pass against the formulas in 64 bits. Bounds, from the roundings: half a step of the type for each
result; half a step of each probability (and of each score's gradient) on its way into a product, added up with
the sizes of what it is multiplied by; scores, exponentials and sums in fp32 with D + 16 steps of 2^-24 of what is added up;
D_i from the rounded result."""
import math

import pytest
import torch
from torch.autograd import forward_ad

import spanqr_amd as sp

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# Half a step of fp16's subnormals, of a result. P goes into its products at 2^7 times at least what it is relative to its row's
# largest (PTINY), and dS times what brings 2 |dO| |V|, the largest ones', to 2^13 at least (2^-25 2 / 2^13 of it). bf16 has
# fp32's exponents, and there the exponential instruction gives 0 below the smallest normal number, 2^-126, as the
# matrix instructions take 0 for bf16's subnormals: a probability of 2^-127 is off by all of it.
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
PTINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -32}
DSTINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -37}


def visible(lq, lk, causal, window):
    i = torch.arange(lq, device="cuda")[:, None] + lk - lq
    j = torch.arange(lk, device="cuda")[None, :]
    seen = torch.ones(lq, lk, dtype=torch.bool, device="cuda")
    if causal:
        seen &= j <= i
        if window:
            seen &= j > i - window
    return seen


def one_head(q, k, v, dout, seen, scale, half=0.0, tiny=0.0, ptiny=0.0, dstiny=0.0):
    """in 64 bits, of one head: (result, bound) of out, dq and this head's part of dk and dv; bounds without the last rounding"""
    q, k, v = q.double(), k.double(), v.double()
    eps = (q.shape[1] + 16) * 2.0 ** -24
    s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    s_err = (eps * (q.abs() @ k.abs().T) * scale).masked_fill(~seen, 0.0)
    if s.shape[1] == 0:
        p, lse = s, torch.full((s.shape[0],), -math.inf, device="cuda", dtype=torch.float64)
    else:
        lse = torch.logsumexp(s, 1)
        p = torch.softmax(s, 1).nan_to_num(0.0)
    # an exponent's error is the score's, and that of its own size; the rows' common part too
    p_err = p * (s_err + s_err.amax(1, keepdim=True) if s.shape[1] else s_err)
    p_err = p_err + p * 2.0 ** -22 * (2.0 + s.abs().masked_fill(~seen, 0.0)) + half * p + ptiny * seen
    o, o_err = p @ v, p_err @ v.abs()
    if dout is None:
        return lse, (o, o_err)
    g = dout.double()
    dp = g @ v.T
    delta = (p * dp).sum(1, keepdim=True)
    # the result as it is rounded, or as it is given
    rounded = half * o.abs() + tiny + o_err
    d_err = (g.abs() * rounded).sum(1, keepdim=True) + eps * (g.abs() * o.abs()).sum(1, keepdim=True)
    ds = p * (dp - delta)
    ds_err = p_err * (dp - delta).abs() + p * (d_err + eps * (g.abs() @ v.abs().T)) + half * ds.abs() + 2.0 ** -126 * seen
    if v.numel() and g.numel():
        ds_err = ds_err + dstiny * seen * float(g.norm(dim=1).max()) * float(v.norm(dim=1).max())
    return lse, (o, o_err), (scale * ds @ k, scale * ds_err @ k.abs()), (scale * ds.T @ q, scale * ds_err.T @ q.abs()), (
        p.T @ g, p_err.T @ g.abs())


def near(got, want, err, what):
    bound = err * 1.001 + HALF[got.dtype] * want.abs() + TINY[got.dtype] + 2.0 ** -22 * err
    bad = ~((got.double() - want).abs() <= bound)   # (NaN is bad)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()}, the worst "
                           f"{float(((got.double() - want).abs() / bound.clamp_min(1e-300))[bad].max())} times its bound, at "
                           f"{bad.nonzero()[0].tolist()}")


def check(q, k, v, dout=None, causal=False, window=None, scale=None, sequences=None, lens=None, **packed):
    """runs the operator and compares; sequences: (first query, end, first key, end) of packed ones; lens: k_lens as numbers"""
    D, H, Hk = q.shape[-1], q.shape[-2], k.shape[-2]
    if lens is not None:
        packed["k_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    small = HALF[q.dtype], TINY[q.dtype], PTINY[q.dtype], DSTINY[q.dtype]
    out, lse = sp.attention(q, k, v, causal=causal, window=window, scale=scale, return_lse=True, **packed)
    grads = [] if dout is None else sp.attention_backward(dout, q, k, v, out, lse, causal=causal, window=window, scale=scale, **packed)
    got = {"out": out}
    got.update(zip(("dq", "dk", "dv"), grads))
    c = D ** -0.5 if scale is None else scale

    def zeros(t):
        return torch.zeros(t.shape, dtype=torch.float64, device="cuda"), torch.zeros(t.shape, dtype=torch.float64, device="cuda")

    want = {n: zeros(t) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v)) if n in got}
    want_lse = torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device="cuda")
    if sequences is None:
        at = [((b,), (b, slice(0, k.shape[1] if lens is None else lens[b]))) for b in range(q.shape[0])]
    else:
        at = [((slice(a, e),), (slice(x, y),)) for a, e, x, y in sequences]
    for qa, ka in at:
        lq, lk = q[qa].shape[0], k[ka].shape[0]
        seen = visible(lq, lk, causal, window)
        for h in range(H):
            hk = h // (H // Hk)
            r = one_head(q[qa][:, h], k[ka][:, hk], v[ka][:, hk], None if dout is None else dout[qa][:, h], seen, c, *small)
            want_lse[qa][:, h] = r[0]
            for n, (value, err), where, head in zip(("out", "dq", "dk", "dv"), r[1:], (qa, qa, ka, ka), (h, h, hk, hk)):
                want[n][0][where][:, head] += value
                want[n][1][where][:, head] += err
    for n, (value, err) in want.items():
        # sums over keys, or over rows, in fp32
        near(got[n], value, err * (1 + 2.0 ** -10), n)
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    scores = float(q.nan_to_num().double().norm(dim=-1).max() * k.nan_to_num().double().norm(dim=-1).max() * c) if q.numel() and k.numel() else 0.0
    assert ((lse.double() - want_lse)[~empty].abs() <= 2.0 ** -20 * (1 + scores)).all()
    return got, lse


def normal(*shape, seed=0, dtype=torch.bfloat16, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (size * torch.randn(*shape, generator=g, device="cuda")).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Sq,Sk,H,Hk,D,causal,window", [
    (1, 1, 1, 1, 1, 8, False, None), (1, 1, 1, 2, 1, 128, True, None), (2, 32, 64, 2, 2, 64, False, None),
    (1, 33, 65, 3, 1, 128, True, None), (2, 100, 100, 4, 2, 64, True, None), (1, 130, 131, 5, 1, 128, True, 7),
    (2, 257, 257, 6, 2, 80, True, 64), (1, 64, 300, 3, 3, 24, False, None), (1, 300, 64, 4, 1, 128, True, None),
    (1, 300, 64, 4, 1, 64, False, None), (1, 200, 70, 1, 1, 72, True, 1), (3, 127, 129, 7, 7, 40, True, None),
    (1, 1000, 1000, 2, 1, 128, True, 100), (1, 700, 700, 2, 2, 64, True, None), (1, 90, 90, 65, 1, 64, True, None),
    (2, 50, 513, 40, 8, 128, True, None),
    # long and few heads: several workgroups to a tile of the gradient
    (1, 600, 500, 8, 1, 64, True, None), (2, 700, 900, 2, 1, 128, False, None), (1, 1100, 1100, 1, 1, 96, True, 130),
    (1, 2000, 130, 3, 1, 32, True, None), (1, 130, 3000, 2, 2, 128, True, None),
    # as many workgroups as make the gradient of K and V take 128 keys each
    (33, 200, 300, 8, 8, 128, True, None), (50, 150, 260, 12, 6, 64, True, 40), (30, 129, 257, 9, 9, 96, False, None)])
def test_batches(cuda, B, Sq, Sk, H, Hk, D, causal, window, dtype):
    q, k, v = normal(B, Sq, H, D, seed=1, dtype=dtype, size=1.5), normal(B, Sk, Hk, D, seed=2, dtype=dtype, size=1.5), normal(
        B, Sk, Hk, D, seed=3, dtype=dtype)
    dout = normal(B, Sq, H, D, seed=4, dtype=dtype)
    got, lse = check(q, k, v, dout, causal, window)
    again = sp.attention_backward(dout, q, k, v, got["out"], lse, causal=causal, window=window)
    assert all(torch.equal(a, got[n]) for a, n in zip(again, ("dq", "dk", "dv")))
    assert torch.equal(sp.attention(q, k, v, causal=causal, window=window), got["out"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Sq,Sk,H,Hk,D,window", [
    (1, 1, 8191, 40, 8, 128, None), (1, 1, 129, 2, 1, 64, None), (3, 1, 1000, 12, 12, 64, None), (1, 5, 4097, 8, 1, 128, None),
    (2, 1, 3000, 8, 2, 128, 300), (1, 2, 640, 3, 3, 48, None), (1, 64, 40000, 1, 1, 64, None)])
def test_tokens_against_a_cache(cuda, B, Sq, Sk, H, Hk, D, window, dtype):
    q, k, v = normal(B, Sq, H, D, seed=1, dtype=dtype, size=1.5), normal(B, Sk, Hk, D, seed=2, dtype=dtype, size=1.5), normal(
        B, Sk, Hk, D, seed=3, dtype=dtype)
    check(q, k, v, causal=True, window=window)
    if window is None and Sq == 1:
        assert torch.equal(sp.attention(q, k, v), sp.attention(q, k, v, causal=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Sq,Sk,H,Hk,D,window,lens", [
    (1, 5000, 16, 2, 128, None, [5000, 1, 0, 2500, 64, 65]), (1, 300, 4, 4, 64, None, [3, 0, 300, 128]), (4, 2000, 8, 1, 80, 100, [2, 1999, 700]),
    (500, 700, 4, 1, 64, None, [700, 0, 333]), (70, 200, 4, 2, 64, None, [200, 70, 13, 0, 129]), (130, 300, 3, 1, 128, 50, [0, 300, 299, 31, 64])])
def test_lengths_of_a_cache(cuda, Sq, Sk, H, Hk, D, window, lens, dtype):
    """what lies behind a sequence's keys is NaN, and neither read nor given a gradient"""
    B = len(lens)
    q, dout = normal(B, Sq, H, D, seed=1, dtype=dtype, size=1.5), normal(B, Sq, H, D, seed=4, dtype=dtype)
    k, v = normal(B, Sk, Hk, D, seed=2, dtype=dtype, size=1.5), normal(B, Sk, Hk, D, seed=3, dtype=dtype)
    for b, n in enumerate(lens):
        k[b, n:] = v[b, n:] = float("nan")
    check(q, k, v, dout, True, window, lens=lens)
    if window is None:
        check(q, k, v, dout, lens=lens)
    # numbers outside 0 to Sk are taken as these
    wild = torch.tensor([-5 if n == 0 else n if n < Sk else Sk + 7 for n in lens], dtype=torch.int32, device=cuda)
    assert torch.equal(sp.attention(q, k, v, k_lens=wild), sp.attention(q, k, v, k_lens=wild.clamp(0, Sk)))


def test_lengths_autograd_and_replays(cuda):
    """k_lens changed between replays, as a cache grows; the gradient through autograd; batch strides"""
    cache = normal(3, 500, 2, 2, 64)
    q = normal(3, 1, 8, 64, seed=5)
    lens = torch.tensor([1, 100, 499], dtype=torch.int32, device=cuda)
    k, v = cache[:, :, 0], cache[:, :, 1]

    def step():
        return sp.attention(q, k, v, causal=True, k_lens=lens)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        graph.replay()
        eager = step()
        assert torch.equal(got, eager)
        for b, n in enumerate(lens.tolist()):
            # (other splits of the keys, so other roundings: two calls, each half a step of the probabilities and of the result,
            # which is below sum p |v|, known to 2 half steps of itself)
            at = q[b:b + 1], k[b:b + 1, :n]
            most = sp.attention(*at, v[b:b + 1, :n].abs()).float()
            assert ((sp.attention(*at, v[b:b + 1, :n]) - eager[b]).float().abs() <= 4.1 * 2.0 ** -8 * most).all()
        lens.add_(1).clamp_(max=500)
    leaf = cache.clone().requires_grad_()
    lens = torch.tensor([1, 0, 77], dtype=torch.int32, device=cuda)
    out, lse = sp.attention(q, leaf[:, :, 0], leaf[:, :, 1], k_lens=lens, return_lse=True)
    out.backward(q)
    _, dk, dv = sp.attention_backward(q, q, k, v, out.detach(), lse, k_lens=lens)
    assert torch.equal(leaf.grad, torch.stack([dk, dv], 2)) and not leaf.grad[1].any() and not leaf.grad[2, 77:].any()


def packed_case(lq, lk, H, Hk, D, dtype, front=0, behind=0):
    """sequences end to end, with rows of no sequence around them, which hold NaN"""
    def starts(n):
        at = [front]
        for x in n:
            at.append(at[-1] + x)
        return at

    qs, ks = starts(lq), starts(lk)
    q, dout = (normal(qs[-1] + behind, H, D, seed=s, dtype=dtype, size=1.5) for s in (1, 2))
    k, v = (normal(ks[-1] + behind, Hk, D, seed=s, dtype=dtype) for s in (3, 4))
    for t, end in ((q, qs[-1]), (dout, qs[-1]), (k, ks[-1]), (v, ks[-1])):
        t[:front] = float("nan")
        t[end:] = float("nan")
    return q, k, v, dout, dict(q_starts=torch.tensor(qs, dtype=torch.int32, device="cuda"),
                               k_starts=torch.tensor(ks, dtype=torch.int32, device="cuda"),
                               sequences=list(zip(qs, qs[1:], ks, ks[1:])))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lq,lk,H,Hk,D,causal,window,front,behind", [
    ([5], [5], 2, 1, 64, True, None, 0, 0), ([100, 1, 0, 300, 64], [100, 1, 0, 300, 64], 4, 2, 128, True, None, 0, 0),
    ([100, 1, 0, 33, 64], [7, 200, 50, 0, 64], 4, 2, 64, True, None, 3, 9),
    ([700, 3, 0, 500], [600, 3, 9, 500], 2, 1, 64, True, None, 5, 7), ([1200], [1200], 1, 1, 128, True, 300, 2, 3),
    ([130, 257, 31], [130, 257, 31], 3, 1, 96, True, 50, 1, 200), ([65, 0, 0, 129], [64, 0, 9, 200], 5, 5, 128, False, None, 0, 1)])
def test_packed(cuda, lq, lk, H, Hk, D, causal, window, front, behind, dtype):
    q, k, v, dout, packed = packed_case(lq, lk, H, Hk, D, dtype, front, behind)
    got, lse = check(q, k, v, dout, causal, window, **packed)
    sequences = packed.pop("sequences")
    # hints change what is launched, not what comes out (but for another number of parts: other sums, which are within the same
    # bounds); too small ones included
    for hints in (dict(max_q=max(lq), max_k=max(lk)), dict(max_q=1, max_k=1), dict(max_q=10 ** 9, max_k=10 ** 9)):
        out, lse2 = sp.attention(q, k, v, causal=causal, window=window, return_lse=True, **packed, **hints)
        split = not torch.equal(out, got["out"])   # (another number of splits: other sums)
        assert not split or (out.double() - got["out"].double()).abs().max() <= 4 * HALF[dtype] * float(v.nan_to_num().abs().max())
        grads = sp.attention_backward(dout, q, k, v, got["out"], lse, causal=causal, window=window, **packed, **hints)
        if not all(torch.equal(g, got[n]) for g, n in zip(grads, ("dq", "dk", "dv"))):
            check(q, k, v, dout, causal, window, sequences=sequences, **packed, **hints)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_tokens(cuda, dtype):
    """one token a request, ragged contexts, an empty one, a request without a token, rows around them"""
    lk = [4000, 1, 0, 700, 63, 64, 65, 2000]
    q, k, v, _, packed = packed_case([1, 1, 1, 1, 1, 0, 1, 3], lk, 16, 2, 128, dtype, 2, 5)
    check(q, k, v, None, True, **packed, max_q=1, max_k=4000)
    check(q, k, v, None, True, **packed)


def test_one_sequence_packed_is_the_batch(cuda):
    q, k, v, dout = (normal(1, 333, h, 64, seed=s) for s, h in ((1, 4), (2, 2), (3, 2), (4, 4)))
    out, lse = sp.attention(q, k, v, causal=True, return_lse=True)
    starts = torch.tensor([0, 333], dtype=torch.int32, device=cuda)
    out2, lse2 = sp.attention(q[0], k[0], v[0], causal=True, q_starts=starts, return_lse=True)
    assert torch.equal(out[0], out2) and torch.equal(lse[0], lse2)
    for a, b in zip(sp.attention_backward(dout, q, k, v, out, lse, causal=True),
                    sp.attention_backward(dout[0], q[0], k[0], v[0], out2, lse2, causal=True, q_starts=starts)):
        assert torch.equal(a[0], b)


def test_strides(cuda):
    """columns of one product, heads before rows, expanded keys, rows that start off 16 bytes, odd offsets: as the same dense ones"""
    B, S, H, Hk, D = 2, 150, 4, 2, 64
    qkv = normal(B, S, (H + 2 * Hk), D, seed=1)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    dout = normal(B, H, S, D, seed=2).transpose(1, 2)

    def run(q, k, v, dout):
        out, lse = sp.attention(q, k, v, causal=True, return_lse=True)
        return (out, lse, *sp.attention_backward(dout, q, k, v, out, lse, causal=True))

    want = run(*(t.contiguous() for t in (q, k, v, dout)))
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, v, dout), want))
    odd = torch.empty(B, S, H, D + 3, dtype=q.dtype, device=cuda)[..., 1:D + 1]
    odd.copy_(q)
    assert all(torch.equal(a, b) for a, b in zip(run(odd, k, v, dout), want))
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    columns = k.transpose(2, 3).contiguous().transpose(2, 3)
    assert all(torch.equal(a, b) for a, b in zip(run(heads_first, columns, v, dout), want))
    k1, v1 = k[:1, :, :1].expand(B, S, Hk, D), v[:1, :, :1].expand(B, S, Hk, D)
    want = run(*(t.contiguous() for t in (q, k1, v1, dout)))
    assert all(torch.equal(a, b) for a, b in zip(run(q, k1, v1, dout), want))
    one = torch.ones((), dtype=q.dtype, device=cuda).expand(B, S, H, D)   # the gradient of a sum
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, v, one), run(q, k, v, one.contiguous())))


def test_sizes_of_scores(cuda):
    """scores far apart, all equal, and beyond what an exponential holds; a row's base that rises late"""
    S, D = 300, 64
    q, k, v, dout = (normal(1, S, 2, D, seed=s) for s in (1, 2, 3, 4))
    check(q * 30, k, v, dout, True)
    check(q * 0, k, v, dout, True)
    check(q, k, v, dout, True, scale=1e-3)
    ramp = torch.linspace(0, 60, S, device=cuda)[None, :, None, None].to(q.dtype)
    check(torch.ones_like(q), torch.ones_like(k) * ramp, v, dout, False, scale=1.0 / D)
    check(torch.ones_like(q), torch.ones_like(k) * ramp.flip(1), v, dout, True, scale=1.0 / D)


@pytest.mark.parametrize("size", [1e-5, 1e-3, 30.0])
def test_sizes_of_gradients(cuda, size):
    """fp16: gradients far below its normal numbers, and large ones against large values, of long rows; heads of other sizes beside"""
    S, D = 1000, 64
    q, k, v, dout = (normal(2, S, h, D, seed=s, dtype=torch.float16) for s, h in ((1, 4), (2, 2), (3, 2), (4, 4)))
    v[:, :, 1] *= 10.0
    dout[1] *= 0.01
    got, _ = check(q, k, v, (dout * size).half(), True)
    if size < 1:
        assert got["dq"].any() and got["dk"].any()
    v[0, 5, 0] = 0.0
    dout[0, 7] = 0.0
    check(q, k, v, (dout * size).half(), False)


def test_nothing_to_do(cuda):
    for B, Sq, Sk in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        q, k, v = normal(B, Sq, 4, 64), normal(B, Sk, 2, 64), normal(B, Sk, 2, 64)
        out, lse = sp.attention(q, k, v, return_lse=True)
        assert out.shape == q.shape and not out.any() and (lse == -math.inf).all()
        dq, dk, dv = sp.attention_backward(q, q, k, v, out, lse)
        assert not dq.any() and not dk.any() and not dv.any() and dk.shape == k.shape
    starts = torch.zeros(1, dtype=torch.int32, device=cuda)   # no sequence at all
    q, k, v = normal(70, 4, 64), normal(9, 2, 64), normal(9, 2, 64)
    out, lse = sp.attention(q, k, v, q_starts=starts, k_starts=starts, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    assert not any(g.any() for g in sp.attention_backward(q, q, k, v, out, lse, q_starts=starts, k_starts=starts))


def test_not_a_number_stays_in_its_sequence(cuda):
    q, k, v, dout, packed = packed_case([70, 70, 70], [70, 70, 70], 2, 1, 64, torch.bfloat16)
    packed.pop("sequences")
    clean = sp.attention(q, k, v, causal=True, **packed)
    v2 = v.clone()
    v2[75] = float("nan")
    out = sp.attention(q, k, v2, causal=True, **packed)
    assert torch.equal(out[:70], clean[:70]) and torch.equal(out[140:], clean[140:]) and torch.isnan(out[75:140]).any()


def test_autograd(cuda):
    q, k, v = (normal(2, 40, h, 16, seed=s).requires_grad_() for s, h in ((1, 4), (2, 2), (3, 2)))
    dout = normal(2, 40, 4, 16, seed=4)
    out, lse = sp.attention(q, k, v, causal=True, return_lse=True)
    assert not lse.requires_grad
    grads = torch.autograd.grad(out, (q, k, v), dout, retain_graph=True)
    want = sp.attention_backward(dout, q, k, v, out, lse, causal=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, want)) and not any(w.requires_grad for w in want)
    only, = torch.autograd.grad(out, k, dout, retain_graph=True)
    assert torch.equal(only, grads[1])
    g, = torch.autograd.grad(out, q, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        g.float().square().sum().backward()
    a, b, c = sp.attention_backward(dout, q, k, v, out, lse, causal=True, need_dkv=False)
    assert torch.equal(a, grads[0]) and b is None and c is None
    a, b, c = sp.attention_backward(dout, q, k, v, out, lse, causal=True, need_dq=False)
    assert a is None and torch.equal(b, grads[1]) and torch.equal(c, grads[2])
    long = normal(1, 900, 1, 64, seed=8)   # (several workgroups to a tile)
    out, lse = sp.attention(long, long, long, return_lse=True)
    both = sp.attention_backward(long, long, long, long, out, lse)
    assert torch.equal(sp.attention_backward(long, long, long, long, out, lse, need_dkv=False)[0], both[0])
    assert all(torch.equal(x, y) for x, y in zip(sp.attention_backward(long, long, long, long, out, lse, need_dq=False)[1:], both[1:]))
    starts = torch.tensor([0, 13, 40], dtype=torch.int32, device=cuda)
    packed = sp.attention(q[0], k[0], v[0], causal=True, q_starts=starts)
    assert torch.autograd.grad(packed.float().sum(), q)[0][1].abs().sum() == 0


def test_gradient_against_differences(cuda):
    """the formula's gradients (which the kernels are compared with above) along directions, in 64 bits"""
    q, k, v, dout = (normal(20, 16, seed=s).double() for s in (1, 2, 3, 4))
    seen = visible(20, 20, True, 6)

    def loss(q, k, v):
        return float((torch.softmax((q @ k.T / 4).masked_fill(~seen, -math.inf), 1) @ v * dout).sum())

    _, _, (dq, _), (dk, _), (dv, _) = one_head(q, k, v, dout, seen, 0.25)
    for i, g in enumerate((dq, dk, dv)):
        d = normal(20, 16, seed=9).double()
        up, down = (loss(*(t + s * 1e-5 * d if j == i else t for j, t in enumerate((q, k, v)))) for s in (1, -1))
        # (the difference's error is of the order of its step squared, 1e-10)
        assert abs((up - down) / 2e-5 - float((g * d).sum())) <= 1e-7 * (1 + float((g * d).abs().sum()))


def test_limits_beyond_the_numbers_of_the_library(cuda):
    """windows and lengths larger than any there are, 64 bits included"""
    q, k, v = normal(1, 70, 2, 16), normal(1, 70, 1, 16, seed=1), normal(1, 70, 1, 16, seed=2)
    want, starts = sp.attention(q, k, v, causal=True), torch.tensor([0, 70], dtype=torch.int32, device=cuda)
    for n in (70, 1 << 31, (1 << 32) + 3, 1 << 63, (1 << 64) + 3):
        assert torch.equal(sp.attention(q, k, v, causal=True, window=n), want), n
        assert torch.equal(sp.attention(q[0], k[0], v[0], causal=True, q_starts=starts, max_q=n, max_k=n), want[0]), n


def test_tangents_are_refused(cuda):
    q, k, v = normal(1, 4, 2, 16), normal(1, 4, 2, 16, seed=1), normal(1, 4, 2, 16, seed=2)
    out, lse = sp.attention(q, k, v, return_lse=True)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(q.clone(), torch.ones_like(q))
        for f in (lambda: sp.attention(d, k, v), lambda: sp.attention(q, d, v), lambda: sp.attention(q, k, d),
                  lambda: sp.attention_backward(d, q, k, v, out, lse)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()


def test_refusals(cuda):
    q, k, v = normal(2, 6, 4, 16), normal(2, 6, 2, 16), normal(2, 6, 2, 16)
    starts = torch.tensor([0, 6], dtype=torch.int32, device=cuda)
    out, lse = sp.attention(q, k, v, return_lse=True)
    for f in (lambda: sp.attention(q[0], k, v), lambda: sp.attention(q, k[:1], v), lambda: sp.attention(q, k, v[:, :5]),
              lambda: sp.attention(q[:, :, :3], k, v), lambda: sp.attention(q[..., :12], k[..., :12], v[..., :12]),
              lambda: sp.attention(q, k[..., :8], v[..., :8]), lambda: sp.attention(q, k, v, window=4),
              lambda: sp.attention(q, k, v, causal=True, window=0), lambda: sp.attention(q, k, v, scale=0.0),
              lambda: sp.attention(q, k, v, scale=float("nan")), lambda: sp.attention(q, k, v, scale=-1.0),
              lambda: sp.attention(q, k, v, q_starts=starts), lambda: sp.attention(q, k, v, max_q=3),
              lambda: sp.attention(q, k, v, k_starts=starts), lambda: sp.attention(q[0], k[0, :5], v[0, :5], q_starts=starts),
              lambda: sp.attention(q[0], k[0], v[0], q_starts=starts, k_starts=starts[:1]),
              lambda: sp.attention(q[0], k[0], v[0], q_starts=starts[:0]),
              lambda: sp.attention(q[0], k[0], v[0], q_starts=starts, max_q=-1),
              lambda: sp.attention(q, k, v, k_lens=starts[:1]), lambda: sp.attention(q, k, v, k_lens=starts.cpu()),
              lambda: sp.attention(q[0], k[0], v[0], q_starts=starts, k_lens=starts[:1]),
              lambda: sp.attention(normal(1, 2, 1, 136), normal(1, 2, 1, 136), normal(1, 2, 1, 136)),
              lambda: sp.attention_backward(q[:1], q, k, v, out, lse), lambda: sp.attention_backward(q, q, k, v, out[:1], lse),
              lambda: sp.attention_backward(q, q, k, v, out, lse[:1])):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: sp.attention(q.float(), k.float(), v.float()), lambda: sp.attention(q, k.half(), v),
              lambda: sp.attention(q[0], k[0], v[0], q_starts=starts.long()), lambda: sp.attention(q, k, v, k_lens=starts.long()),
              lambda: sp.attention_backward(q.half(), q, k, v, out, lse),
              lambda: sp.attention_backward(q, q, k, v, out, lse.half()), lambda: sp.attention(q.cpu(), k.cpu(), v.cpu())):
        with pytest.raises(TypeError):
            f()


def test_graph_and_streams(cuda):
    """captured, with inputs and starts changed between replays and eager calls between them"""
    q, k, v, dout, packed = packed_case([100, 60, 40], [100, 60, 40], 4, 2, 64, torch.bfloat16)
    starts = packed["q_starts"]
    token, cache, values = normal(1, 1, 8, 64), normal(1, 2000, 2, 64, seed=5), normal(1, 2000, 2, 64, seed=6)

    def step():
        out, lse = sp.attention(q, k, v, causal=True, q_starts=starts, return_lse=True)
        return (out, lse, *sp.attention_backward(dout, q, k, v, out, lse, causal=True, q_starts=starts),
                sp.attention(token, cache, values))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i, at in enumerate(([0, 100, 160, 200], [0, 1, 1, 200], [0, 0, 150, 170], [0, 100, 160, 200])):
        starts.copy_(torch.tensor(at, dtype=torch.int32))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        if at[1] == 100:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def lengths(n, most, seed, every=3):
    """n lengths up to `most`, some of them 0"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(0, most + 1, (n,), generator=g)
    x[torch.randint(0, every, (n,), generator=g) == 0] = 0
    return x.tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,most,long,H,Hk,D,window,front,behind", [
    (70, 200, 700, 2, 1, 64, None, 5, 900), (130, 40, 1500, 3, 1, 128, 50, 0, 3), (20, 300, 0, 10, 2, 40, None, 400, 0),
    (4200, 3, 260, 1, 1, 16, None, 1, 2)])
def test_many_packed_without_hints(cuda, n, most, long, H, Hk, D, window, front, behind, dtype):
    """sequences of unlike lengths in one list of tiles, one long one among them, with hints and without"""
    lq = lengths(n, most, seed=1)
    lk = lengths(n, most, seed=2)
    lq[n // 2], lk[n // 2] = lq[n // 2] + long, lk[n // 2] + long
    q, k, v, dout, packed = packed_case(lq, lk, H, Hk, D, dtype, front, behind)
    got, lse = check(q, k, v, dout, True, window, **packed)
    sequences = packed.pop("sequences")
    hints = dict(max_q=max(lq), max_k=max(lk))
    out, lse2 = sp.attention(q, k, v, causal=True, window=window, return_lse=True, **packed, **hints)
    if not (torch.equal(out, got["out"]) and torch.equal(lse, lse2)):   # (another number of parts)
        check(q, k, v, dout, True, window, sequences=sequences, **packed, **hints)


def test_more_tiles_than_workgroups(cuda):
    """a launch takes fewer than 2^24 workgroups; 2^24 tiles are gone over by 2^23"""
    B = (1 << 23) - 1
    q, k, v = normal(1, 1, 129, 8, seed=1), normal(1, 4, 1, 8, seed=2), normal(1, 4, 1, 8, seed=3)
    dout = normal(1, 1, 129, 8, seed=4)

    def all_of(t):
        return t.expand(B, *t.shape[1:])

    want, lse = sp.attention(q, k, v, return_lse=True)
    out = sp.attention(all_of(q), all_of(k), all_of(v))
    assert torch.equal(out[0], want[0]) and not (out != want).any()
    del out
    dq, _, _ = sp.attention_backward(all_of(dout), all_of(q), all_of(k), all_of(v), all_of(want), all_of(lse), need_dkv=False)
    want, _, _ = sp.attention_backward(dout, q, k, v, want, lse)
    assert torch.equal(dq[0], want[0]) and not (dq != want).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sum_of_many_alike(cuda, dtype):
    """65536 keys that are not split, all but the first 64 with one score (a head's own), on either side of the sum's base. Sums
    over a tile's 32 keys a lane, then over 1024 tiles, of half a step of fp32 (2^-24) each; a score's, its exponential's and lse's own
    roundings 2^-20 of their sizes."""
    Lk, H = 65536, 256
    scores = torch.linspace(-4.0, 5.4, H, device=cuda).to(dtype)
    k = torch.zeros(1, Lk, H, 8, dtype=dtype, device=cuda)
    k[0, 64:, :, 0] = scores
    q = torch.zeros(1, 1, H, 8, dtype=dtype, device=cuda)
    q[..., 0] = 1.0
    v = torch.ones(1, 1, H, 8, dtype=dtype, device=cuda).expand(1, Lk, H, 8)
    out, lse = sp.attention(q, k, v, scale=1.0, return_lse=True)
    want = torch.log(64.0 + (Lk - 64) * scores.double().exp())
    bound = (Lk // 64 + 33) * 2.0 ** -24 + 2.0 ** -20 * (1.0 + scores.double().abs())
    assert ((lse[0, 0].double() - want).abs() <= bound).all()
    assert (out.double() - 1.0).abs().max() <= 4 * HALF[dtype]


def test_long_cache_with_heads_in_front(cuda):
    """keys and values as [heads, rows, D] caches whose heads are 2^24 elements and more apart are read as they lie"""
    S = (1 << 24) // 64 + 1
    keys, values = normal(2, S, 64, seed=1), normal(2, S, 64, seed=2)
    k, v = keys.transpose(0, 1)[None], values.transpose(0, 1)[None]
    assert k.stride(2) > 1 << 24
    q = normal(1, 1, 8, 64, seed=3)
    want = sp.attention(q, k.contiguous(), v.contiguous())
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = sp.attention(q, k, v)
    assert torch.cuda.max_memory_allocated() - before < 16 << 20   # (a copy of the keys is 64 MB)
    assert torch.equal(got, want)
    k, v, q, dout = k[:, -200:], v[:, -200:], normal(1, 100, 4, 64, seed=4), normal(1, 100, 4, 64, seed=5)
    got, lse = sp.attention(q, k, v, causal=True, return_lse=True)
    want = sp.attention_backward(dout, q, k.contiguous(), v.contiguous(), got, lse, causal=True)
    assert torch.equal(got, sp.attention(q, k.contiguous(), v.contiguous(), causal=True))
    assert all(torch.equal(a, b) for a, b in zip(sp.attention_backward(dout, q, k, v, got, lse, causal=True), want))


@pytest.mark.parametrize("own_keys", [False, True])
def test_packed_autograd(cuda, own_keys):
    """the starts as they are kept for the backward pass: bit by bit what attention_backward gives"""
    starts = [3, 16, 16, 40, 70]
    others = [0, 30, 41, 41, 90] if own_keys else starts
    qs, ks = (torch.tensor(s, dtype=torch.int32, device=cuda) for s in (starts, others))
    how = dict(causal=True, window=20, q_starts=qs, **(dict(k_starts=ks) if own_keys else {}))
    q, dout = normal(75, 4, 32, seed=1).requires_grad_(), normal(75, 4, 32, seed=4)
    k, v = (normal(93 if own_keys else 75, 2, 32, seed=s).requires_grad_() for s in (2, 3))
    out, lse = sp.attention(q, k, v, return_lse=True, **how)
    got = torch.autograd.grad(out, (q, k, v), dout)
    want = sp.attention_backward(dout, q, k, v, out, lse, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert got[0][3:16].any() and not got[0][:3].any() and not got[0][70:].any()
    # one sequence alone, as a batch of one
    first = [t.detach() for t in (q[3:16], k[others[0]:others[1]], v[others[0]:others[1]])]
    alone, lse = sp.attention(*(t[None] for t in first), causal=True, window=20, return_lse=True)
    assert torch.equal(alone[0], out[3:16])
    dq, dk, dv = sp.attention_backward(dout[None, 3:16], *(t[None] for t in first), alone, lse, causal=True, window=20)
    assert torch.equal(dq[0], got[0][3:16]) and torch.equal(dk[0], got[1][others[0]:others[1]]) and torch.equal(dv[0], got[2][others[0]:others[1]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_parts_in_graphs_and_on_streams(cuda, dtype):
    """gradients whose tiles several workgroups share, a batch's and those of a list of packed sequences: captured, with inputs and
    starts changed between replays and eager calls between them; and two streams at once, each with a workspace of its own"""
    L = 2000
    x = [normal(L, h, 64, seed=s, dtype=dtype) for s, h in ((1, 2), (2, 1), (3, 1), (4, 2))]
    starts = torch.arange(0, L + 1, 50, dtype=torch.int32, device=cuda)

    def batch(q, k, v, dout):
        q, k, v, dout = (t[None, :900] for t in (q, k, v, dout))
        out, lse = sp.attention(q, k, v, causal=True, return_lse=True)
        return (out, lse, *sp.attention_backward(dout, q, k, v, out, lse, causal=True))

    def packed(q, k, v, dout):
        out, lse = sp.attention(q, k, v, causal=True, q_starts=starts, return_lse=True)
        return (out, lse, *sp.attention_backward(dout, q, k, v, out, lse, causal=True, q_starts=starts))

    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    first = batch(*x) + packed(*x)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s):
            a = batch(*x)
        with torch.cuda.stream(t):
            b = packed(*x)
        torch.cuda.synchronize()
        assert all(torch.equal(u, w) for u, w in zip(a + b, first))
    graphs = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graphs[0]):
        a = batch(*x)
    with torch.cuda.graph(graphs[1]):
        b = packed(*x)
    for i, at in enumerate((None, [0] * 20 + [L] * 21, [7] * 3 + list(range(10, 1910, 50)), None)):
        starts.copy_(torch.arange(0, L + 1, 50) if at is None else torch.tensor(at))
        for u in x:
            u.neg_()
        for graph in graphs:
            graph.replay()
        eager = batch(*x) + packed(*x)
        torch.cuda.synchronize()
        assert all(torch.equal(u, w) for u, w in zip(a + b, eager)), i
    assert all(torch.equal(u, w) for u, w in zip(eager, first))
