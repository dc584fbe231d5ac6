"""examples/train_block.py: attention, block_norm, dropout, rms_norm and the loss together, their gradients against the same
model in 64 bits, and the steps' invariants"""
import importlib.util
import math
import os

import pytest
import torch

from conftest import ROOT
from test_gpu_block import kept

pytestmark = pytest.mark.gpu


def load():
    spec = importlib.util.spec_from_file_location("train_block", os.path.join(ROOT, "examples", "train_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def norm(x, w):
    return x * ((x * x).mean(-1, keepdim=True) + 1e-6).rsqrt() * w


def in_64_bits(m, model, tokens, targets, starts, seed):
    """the loss and the gradients of model.parameters(), in 64 bits throughout"""
    P = [p.detach().double().requires_grad_() for p in model.parameters()]
    embed, head, norms, W = P[0], P[1], P[2:2 + len(model.norms)], P[2 + len(model.norms):]
    H, K, D, n = model.heads, model.key_heads, model.D, len(tokens)
    factor = 65536 / (65536 - round(65536 * m.P))

    def drop(x, index):
        return x * kept(*x.shape, m.P, seed, index) * factor

    h = drop(embed[tokens], 0)
    y = norm(h, norms[0])
    bounds = starts.tolist()
    for i in range(len(W) // 4):
        t = (y @ W[4 * i].T).view(n, H + 2 * K, D)
        rows = []
        for a, e in zip(bounds, bounds[1:]):
            q, k, v = t[a:e, :H], t[a:e, H:H + K].repeat_interleave(H // K, 1), t[a:e, H + K:].repeat_interleave(H // K, 1)
            s = (q.transpose(0, 1) @ k.permute(1, 2, 0)) * D ** -0.5
            s = s.masked_fill(torch.ones(e - a, e - a, device="cuda").triu(1).bool(), -math.inf)
            rows.append((torch.softmax(s, 2) @ v.transpose(0, 1)).transpose(0, 1).reshape(e - a, H * D))
        n1, n2, n3, n4 = norms[4 * i + 1:4 * i + 5]
        h = h + m.SCALE * drop(norm(torch.cat(rows) @ W[4 * i + 1].T, n1), 2 * i + 1)
        y = norm(h, n2)
        value, gate = (y @ W[4 * i + 2].T).chunk(2, 1)
        h = h + m.SCALE * drop(norm(value @ W[4 * i + 3].T, n3) * torch.nn.functional.silu(gate), 2 * i + 2)
        y = norm(h, n4)
    loss = torch.nn.functional.cross_entropy(y @ head.T, targets)
    return loss.detach(), torch.autograd.grad(loss, P)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients(cuda, dtype):
    m = load()
    model = m.Model(vocab=60, width=128, heads=4, key_heads=2, rank=32, layers=2, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(3)
    lengths = [70, 1, 0, 130, 33]
    tokens, targets, starts = m.texts(g, 60, lengths)
    loss = m.gradients(model, tokens, targets, starts, max(lengths), seed=17)
    want, grads = in_64_bits(m, model, tokens, targets, starts, 17)
    # Some thirty roundings to the type lie between a weight and the loss and back, each of half a step at most and
    # independent of each other: their root sum of squares is below 6 half steps of what a gradient is made of, and
    # norms and the softmax pass on at most a few times what they get. 32 half steps of the gradient as a whole.
    half = torch.finfo(dtype).eps / 2
    assert abs(float(loss) - float(want)) <= 32 * half * float(want)
    for i, (p, w) in enumerate(zip(model.parameters(), grads)):
        off = float((p.grad.double() - w).norm() / w.norm())
        assert off <= 32 * half, (i, list(p.shape), off)
    again = m.gradients(model, tokens, targets, starts, max(lengths), seed=17)
    assert torch.equal(loss, again)
    assert not torch.equal(loss, m.gradients(model, tokens, targets, starts, max(lengths), seed=18))


def test_steps(cuda):
    m = load()
    model = m.Model(vocab=40, width=128, rank=32, layers=1)
    g = torch.Generator(device="cuda").manual_seed(4)
    for i in range(3):
        tokens, targets, starts = m.texts(g, 40, [100, 57, 1])
        loss, grad_norm = m.step(model, tokens, targets, starts, 100, seed=i)
        assert math.isfinite(float(loss)) and float(grad_norm) > 0.0
    for V, U, W in zip(model.V, model.U, model.W):
        # orth's own bound
        assert float((V.double().T @ V.double() - torch.eye(32, device=cuda, dtype=torch.float64)).abs().max()) <= 2e-7
        assert torch.equal(W, (U @ V.T).to(W.dtype))
