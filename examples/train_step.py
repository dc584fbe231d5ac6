"""A small language model trained with this library's operators, from the loss to orth:

    python examples/train_step.py --steps 60

Every layer's weight is W = U V^T with orthonormal V, as TTF keeps its layers. One step is

  forward     rms_norm of the residual stream before each layer and before the head
  loss        linear_cross_entropy_grad: the loss and its gradients, without logits in memory
  backward    autograd through the layers; rms_norm brings its own backward
  clipping    clip_grad_norm: the 16-bit gradients, clipped by their global norm, as 32-bit copies
  optimizer   u = the normalised gradient; X = V (U^T U) + u^T U -> orth_many -> the layers' new V, and U = (W + u) V

on random tokens that follow a rule (the next token is a fixed permutation of this one, but for some noise).
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from spanqr_amd import clip_grad_norm, linear_cross_entropy_grad, orth, orth_many, rms_norm  # noqa: E402


class Model:
    def __init__(self, vocab=2000, width=256, rank=64, layers=2, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape):
            return torch.randn(*shape, generator=g, device=device)

        self.embed = (normal(vocab, width)).bfloat16().requires_grad_()
        self.head = (normal(vocab, width) * width ** -0.5).bfloat16().requires_grad_()
        self.norms = [torch.ones(width, device=device, dtype=torch.bfloat16, requires_grad=True) for _ in range(layers + 1)]
        self.V = [orth(normal(width, rank)) for _ in range(layers)]
        self.U = [normal(width, rank) * rank ** -0.5 for _ in range(layers)]
        self.W = [None] * layers
        self.refresh()

    def refresh(self):
        for i, (U, V) in enumerate(zip(self.U, self.V)):
            self.W[i] = (U @ V.T).bfloat16().requires_grad_()

    def parameters(self):
        return [self.embed, self.head, *self.norms, *self.W]

    def hidden(self, tokens):
        """the normed stream before the head"""
        out, stream = self.embed[tokens], None
        for w, W in zip(self.norms, self.W):
            if stream is None:
                stream, y = out, rms_norm(out, w)
            else:
                y, stream = rms_norm(out, w, residual=stream)
            out = torch.nn.functional.silu(y) @ W.T
        return rms_norm(out, self.norms[-1], residual=stream)[0]


def step(model, tokens, targets, rate=0.02, max_norm=1.0):
    """one training step; the loss and the gradients' norm as tensors on the device"""
    params = model.parameters()
    for p in params:
        p.grad = None
    h = model.hidden(tokens)
    loss, dh, model.head.grad = linear_cross_entropy_grad(h, model.head, targets)
    h.backward(dh)
    grads = [p.grad for p in params]
    clipped = [torch.empty(g.shape, dtype=torch.float32, device=g.device) for g in grads]
    norm = clip_grad_norm(grads, max_norm, out=clipped)
    with torch.no_grad():
        plain = len(params) - len(model.W)
        for p, g in zip(params[:plain], clipped):
            p -= (rate * g / (g.square().mean().sqrt() + 1e-12)).to(p.dtype)
        us = [-0.2 * rate * g / (g.square().mean().sqrt() + 1e-12) for g in clipped[plain:]]
        news = orth_many([V @ (U.T @ U) + u.T @ U for U, V, u in zip(model.U, model.V, us)])
        model.U = [U @ (V.T @ N) + u @ N for U, V, N, u in zip(model.U, model.V, news, us)]
        model.V = news
    model.refresh()
    return loss, norm


def train(steps=60, tokens=2048, vocab=2000, ignored=0.05, seed=0, report=None, **sizes):
    """the losses of `steps` steps"""
    model = Model(vocab=vocab, seed=seed, **sizes)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    rule = torch.randperm(vocab, generator=g, device="cuda")
    losses = []
    for i in range(steps):
        x = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
        y = rule[x]
        y = torch.where(torch.rand(tokens, generator=g, device="cuda") < ignored, torch.full_like(y, -100), y)
        loss, norm = step(model, x, y)
        losses.append(loss)
        if report is not None and (i % report == 0 or i == steps - 1):
            print(f"step {i}: loss {float(loss):.4f}, gradient norm {float(norm):.4f}", flush=True)
    return [float(v) for v in losses]


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--vocab", type=int, default=2000)
    args = ap.parse_args()
    train(args.steps, args.tokens, args.vocab, report=10)


if __name__ == "__main__":
    main()
