"""grad_norm and clip_grad_norm against torch in 64 bits. Squares and sums are in 64 bits, so the norm is the 64-bit one
rounded once (2^-24, and 2^-40 for the order of the sums); a clipped element is g times a factor that is rounded once,
rounded again as a product and once to its type."""
import math

import pytest
import torch

import spanqr_amd as sp

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
LISTS = {
    "one element": [(1,)],
    "small": [(3,), (1, 7), (2, 2, 2)],
    "chunks": [(8191,), (8192,), (8193,), (3 * 8192 + 5,)],
    "empty among them": [(0,), (5, 0), (100, 33), (0,), (17,)],
    "many": [(1 + (i * 37) % 101, 1 + i % 13) for i in range(500)],
    "layers": [(768, 512), (2048, 512), (768,)] * 3,
    "a table and one": [(64,)] * 113,
    "a table": [(65,)] * 112,
}


def make(shapes, dtype, seed, scale=0.01):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(scale * torch.randn(*s, generator=g, device="cuda")).to(dtype) for s in shapes]


def norm_of(ts):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))


def check_norm(got, want):
    assert got.dtype == torch.float32 and got.shape == () and got.device.type == "cuda"
    assert abs(float(got) - want) <= want * (E + 2.0 ** -40), (float(got), want)


def check_clipped(outs, grads, max_norm, want):
    f = min(1.0, max_norm / want) if want else 1.0
    for o, g in zip(outs, grads):
        v = g.double() * f
        assert o.shape == g.shape
        d = (o.double() - v).abs()
        assert bool((d <= v.abs() * (2.1 * E + U[o.dtype]) + TINY[o.dtype]).all()), float(d.max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(LISTS))
def test_norm_and_clip(cuda, name, dtype):
    print(f"clip {name} {dtype}", flush=True)
    grads = make(LISTS[name], dtype, 1)
    was = [g.clone() for g in grads]
    want = norm_of(grads)
    check_norm(sp.grad_norm(grads), want)
    for out_dtype in DTYPES:
        outs = [torch.full(g.shape, 7.0, dtype=out_dtype, device=cuda) for g in grads]
        check_norm(sp.clip_grad_norm(grads, 0.3 * want, out=outs), want)
        check_clipped(outs, was, 0.3 * want, want)
        sp.clip_grad_norm(grads, 2 * want, out=outs)        # within: copies
        assert all(torch.equal(o, w.to(out_dtype)) for o, w in zip(outs, was))
    assert all(torch.equal(g, w) for g, w in zip(grads, was))   # read only
    check_norm(sp.clip_grad_norm(grads, 2 * want), want)
    assert all(torch.equal(g, w) for g, w in zip(grads, was))   # in place and within: untouched
    check_norm(sp.clip_grad_norm(grads, 0.3 * want), want)
    check_clipped(grads, was, 0.3 * want, want)


def test_mixed_types_and_odd_starts(cuda):
    flat = make([(100000,)], torch.bfloat16, 2)[0]
    at, grads = 1, []
    for n in (1, 2, 3, 1000, 8192, 777, 20000):
        grads.append(flat[at:at + n])
        at += n
    grads += make([(50, 50)], torch.float32, 3) + make([(333,)], torch.float16, 4)
    was = flat.clone()
    want = norm_of(grads)
    check_norm(sp.grad_norm(grads), want)
    before = [g.clone() for g in grads]
    sp.clip_grad_norm(grads, 0.1 * want)
    check_clipped(grads, before, 0.1 * want, want)
    assert torch.equal(flat[0], was[0]) and torch.equal(flat[at:], was[at:])   # nothing beside them


@pytest.mark.parametrize("dtype", DTYPES)
def test_orders_and_strides(cuda, dtype):
    a, b, c = make([(40, 60), (10, 20, 30), (50, 70)], dtype, 5)
    views = [a.T, b.permute(2, 0, 1), c[:, 3:40], c[::2, 45:], a[7:8]]
    for v in views:
        w = v.clone()
        want = norm_of([v])
        check_norm(sp.grad_norm(v), want)
        out = torch.empty(v.shape, dtype=torch.float32, device=cuda)      # rows, whatever the gradient's order
        sp.clip_grad_norm([v], 0.5 * want, out=[out])
        check_clipped([out], [w], 0.5 * want, want)
        o2 = torch.zeros(*v.shape[:-1], 2 * v.shape[-1], dtype=dtype, device=cuda)[..., ::2]
        sp.clip_grad_norm([v], 0.5 * want, out=[o2])
        check_clipped([o2], [w], 0.5 * want, want)
        sp.clip_grad_norm([v], 0.5 * want)
        check_clipped([v], [w], 0.5 * want, want)
    whole = make([(50, 70)], dtype, 6)[0]
    kept = whole.clone()
    sp.clip_grad_norm([whole[:, 3:40]], 1e-3)
    assert torch.equal(whole[:, :3], kept[:, :3]) and torch.equal(whole[:, 40:], kept[:, 40:])


def test_ranges(cuda):
    """squares beyond and below float32's range, infinities, NaN, zeros"""
    for scale in (1e30, 1e-30):
        g = make([(3000,), (17,)], torch.float32, 7, scale)
        want = norm_of(g)
        check_norm(sp.grad_norm(g), want)
        w = [t.clone() for t in g]
        sp.clip_grad_norm(g, 0.25 * want)
        check_clipped(g, w, 0.25 * want, want)
    g = make([(3000,), (17,)], torch.float32, 8)
    g[1][3] = float("inf")
    assert float(sp.grad_norm(g)) == float("inf")
    out = [torch.empty_like(t) for t in g]
    assert float(sp.clip_grad_norm(g, 1.0, out=out)) == float("inf")
    assert not out[0].any() and torch.isnan(out[1][3]) and not out[1][:3].any()
    g[1][3] = float("nan")
    assert math.isnan(float(sp.clip_grad_norm(g, 1.0, out=out)))
    assert torch.isnan(out[0]).all() and torch.isnan(out[1]).all()
    z = [torch.zeros(10, device=cuda)]
    assert float(sp.clip_grad_norm(z, 0.0)) == 0.0 and not z[0].any()
    g = make([(100,)], torch.float32, 9)
    sp.clip_grad_norm(g, 0.0)
    assert not g[0].any()


def test_nothing(cuda):
    assert float(sp.grad_norm([])) == 0.0 and float(sp.clip_grad_norm([], 1.0)) == 0.0
    assert float(sp.grad_norm([torch.empty(0, device=cuda)])) == 0.0
    assert float(sp.clip_grad_norm([torch.empty(0, 3, device=cuda)], 1.0)) == 0.0


def test_refusals(cuda):
    g = make([(4, 4)], torch.float32, 10)
    for bad in (lambda: sp.clip_grad_norm(g, -1.0), lambda: sp.clip_grad_norm(g, float("nan")),
                lambda: sp.clip_grad_norm(g, 1.0, out=[]), lambda: sp.clip_grad_norm(g, 1.0, out=[g[0][:3]]),
                lambda: sp.clip_grad_norm([g[0][:1].expand(4, 4)], 1.0)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: sp.grad_norm([g[0].double()]), lambda: sp.grad_norm([g[0].cpu()]),
                lambda: sp.clip_grad_norm(g, 1.0, out=[g[0].int()])):
        with pytest.raises(TypeError):
            bad()


def test_graph_and_repeats(cuda):
    grads = make(LISTS["many"], torch.bfloat16, 11)
    outs = [torch.empty(g.shape, dtype=torch.float32, device=cuda) for g in grads]
    norm = sp.clip_grad_norm(grads, 0.05, out=outs)
    eager = [norm] + [o.clone() for o in outs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sp.clip_grad_norm(grads, 0.05, out=outs)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        captured = sp.clip_grad_norm(grads, 0.05, out=outs)
    for rep in range(3):
        captured.zero_()
        for o in outs:
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([captured] + outs, eager)), rep
        assert torch.equal(sp.grad_norm(grads), norm)
