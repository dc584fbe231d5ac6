"""What autograd may not overlook in the training operators: gradients of gradients, tangents of forward-mode
differentiation, tensors that are written in place"""
import pytest
import torch
from torch.autograd import forward_ad

import spanqr_amd as sp

pytestmark = pytest.mark.gpu


def loss_inputs(N=6, H=16, V=40, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(N, H, generator=g, device="cuda").to(dtype).requires_grad_()
    W = (0.3 * torch.randn(V, H, generator=g, device="cuda")).to(dtype).requires_grad_()
    return x, W, torch.randint(0, V, (N,), generator=g, device="cuda")


def norm_inputs(rows=5, D=40, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(2)
    x, r = (torch.randn(rows, D, generator=g, device="cuda").to(dtype).requires_grad_() for _ in range(2))
    return x, torch.ones(D, device="cuda", dtype=dtype, requires_grad=True), r


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_is_not_differentiated_twice(cuda, reduction):
    x, W, t = loss_inputs()
    loss = sp.linear_cross_entropy(x, W, t, reduction=reduction).sum()
    plain = torch.autograd.grad(loss, (x, W), retain_graph=True)
    gx, gw = torch.autograd.grad(loss, (x, W), create_graph=True)
    assert torch.equal(gx, plain[0]) and torch.equal(gw, plain[1])
    for g in (gx, gw):
        with pytest.raises(RuntimeError, match="differentiated again"):
            (loss + g.float().square().sum()).backward(retain_graph=True)
    # one of the two alone
    W2 = W.detach()
    loss = sp.linear_cross_entropy(x, W2, t, reduction=reduction).sum()
    gx, = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        gx.float().square().sum().backward()


@pytest.mark.parametrize("residual", [False, True])
def test_norm_is_not_differentiated_twice(cuda, residual):
    x, w, r = norm_inputs()
    y = sp.rms_norm(x, w, residual=r)[0] if residual else sp.rms_norm(x, w)
    loss = y.float().square().sum()
    inputs = (x, w, r) if residual else (x, w)
    plain = torch.autograd.grad(loss, inputs, retain_graph=True)
    grads = torch.autograd.grad(loss, inputs, create_graph=True)
    for g, p in zip(grads, plain):
        assert torch.equal(g, p)
        with pytest.raises(RuntimeError, match="differentiated again"):
            (loss + g.float().square().sum()).backward(retain_graph=True)


def test_create_graph_alone_is_fine(cuda):
    """steps that record the backward pass and do not use what it recorded, with the gradients added up and set to zero"""
    x, W, t = loss_inputs()
    w = torch.ones(16, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    for _ in range(2):
        loss = sp.linear_cross_entropy(sp.rms_norm(x, w), W, t)
        loss.backward(create_graph=True)
    for p in (x, W, w):
        assert p.grad.requires_grad
        p.grad = p.grad.detach()
    twice = [p.grad.clone() for p in (x, W, w)]
    for p in (x, W, w):
        p.grad.zero_()
    for _ in range(2):
        sp.linear_cross_entropy(sp.rms_norm(x, w), W, t).backward()
    assert all(torch.equal(p.grad, v) for p, v in zip((x, W, w), twice))


def test_tangents_are_refused(cuda):
    x, W, t = loss_inputs()
    x, W = x.detach(), W.detach()
    h, w, r = (v.detach() for v in norm_inputs())
    calls = [(x, lambda d: sp.linear_cross_entropy(d, W, t)), (W, lambda d: sp.linear_cross_entropy(x, d, t)),
             (x, lambda d: sp.linear_cross_entropy_grad(d, W, t)),
             (torch.ones(len(t), device=cuda), lambda d: sp.linear_cross_entropy_grad(x, W, t, row_weight=d)),
             (torch.ones((), device=cuda), lambda d: sp.linear_cross_entropy_grad(x, W, t, grad_scale=d)),
             (h, lambda d: sp.rms_norm(d, w)), (w, lambda d: sp.rms_norm(h, d)), (r, lambda d: sp.rms_norm(h, w, residual=d)),
             (h, lambda d: sp.rms_norm(d, w, quant="int8")), (r, lambda d: sp.rms_norm_backward(d, h, w)),
             (r, lambda d: sp.rms_norm_backward(r, h, w, dh=d)), (h, lambda d: sp.grad_norm([r, d])),
             (h, lambda d: sp.clip_grad_norm(d, 1.0)), (h, lambda d: sp.clip_grad_norm([r.clone()], 1.0, out=[d]))]
    for v, call in calls:
        want = call(v.clone())
        with forward_ad.dual_level():
            assert torch.equal(*(c[0] if isinstance(c, tuple) else c for c in (call(v.clone()), want)))   # no tangent
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(forward_ad.make_dual(v.clone(), torch.ones_like(v)))


@pytest.mark.parametrize("strided", [False, True])
def test_clipping_is_seen(cuda, strided):
    """a tensor that autograd keeps and that is clipped in place, or written as out, is not the one it kept"""
    def kept():
        a = torch.ones(6, 8, device=cuda, requires_grad=True)
        b = a * 3.0
        c = b.square().sum()         # keeps b
        b = b.detach()
        return b[:, ::2] if strided else b, c

    b, c = kept()
    sp.grad_norm([b])                # reads alone
    c.backward()
    for write in (lambda t: sp.clip_grad_norm([t], 1.0), lambda t: sp.clip_grad_norm([torch.ones_like(t)], 1.0, out=[t])):
        b, c = kept()
        was = b._version
        write(b)
        assert b._version > was
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            c.backward()
    g = torch.ones(5, device=cuda)
    was = g._version
    sp.clip_grad_norm([g], 1.0, out=[torch.empty_like(g)])
    assert g._version == was
    with torch.inference_mode():     # such tensors have no version
        sp.clip_grad_norm([torch.ones(5, device=cuda)], 1.0)


@pytest.mark.parametrize("strided", [False, True])
def test_clipping_records_nothing(cuda, strided):
    """gradients that require a gradient (of a recorded backward pass, or leaves) are clipped as others are, in any order"""
    whole = torch.ones(6, 8, device=cuda)
    leaf = (whole[:, ::2] if strided else whole).requires_grad_()
    sp.clip_grad_norm([leaf], 1.0)
    assert leaf.is_leaf and abs(float(leaf.detach().norm()) - 1.0) < 1e-6
    a = torch.ones(6, 8, device=cuda, requires_grad=True)
    b = (a * 1.0)[:, ::2] if strided else a * 1.0
    sp.clip_grad_norm([b], 1.0)
    assert abs(float(b.detach().norm()) - 1.0) < 1e-6
    b.sum().backward()               # as before: the factor is no part of it
    assert float(a.grad.sum()) == b.numel()
