"""One training step of a small transformer with this library's operators, on texts packed end to end:

    python examples/train_block.py --steps 40

A layer is attention and a gated feed-forward block; each hands its result on through block_norm: normed, dropped out,
added to the residual stream at half its size, and the stream normed for the next block. The weights of the products are
W = U V^T with orthonormal V, and orth_many finds the new V from the clipped gradients, as in train_step.py.

  forward     rms_norm of the embedding, then per layer: attention, block_norm, feed-forward, block_norm with the gate
  loss        linear_cross_entropy_grad
  backward    autograd; attention and block_norm bring their own
  optimizer   clip_grad_norm, then X = V (U^T U) + u^T U -> orth_many -> the layers' new V, and U = (W + u) V
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from spanqr_amd import (attention, block_norm, clip_grad_norm, dropout, linear_cross_entropy_grad, orth, orth_many,  # noqa: E402
                        rms_norm)

P = 0.1        # dropout
SCALE = 0.5    # of what a block adds to the stream


class Model:
    def __init__(self, vocab=500, width=128, heads=4, key_heads=2, rank=32, layers=2, seed=0, dtype=torch.bfloat16, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape):
            return torch.randn(*shape, generator=g, device=device)

        self.heads, self.key_heads, self.dtype = heads, key_heads, dtype
        self.D = width // heads
        self.embed = normal(vocab, width).to(dtype).requires_grad_()
        self.head = (normal(vocab, width) * width ** -0.5).to(dtype).requires_grad_()
        self.norms = [torch.ones(width, device=device, dtype=dtype, requires_grad=True) for _ in range(4 * layers + 1)]
        # per layer: q, k and v in one; the result's product; the feed-forward block's value and gate, and its result's
        outs = [(heads + 2 * key_heads) * self.D, width, 2 * width, width] * layers
        self.V = [orth(normal(width, rank)) for _ in outs]
        self.U = [normal(n, rank) * rank ** -0.5 for n in outs]
        self.W = [None] * len(outs)
        self.refresh()

    def refresh(self):
        for i, (U, V) in enumerate(zip(self.U, self.V)):
            self.W[i] = (U @ V.T).to(self.dtype).requires_grad_()

    def parameters(self):
        return [self.embed, self.head, *self.norms, *self.W]

    def hidden(self, tokens, starts, longest, seed):
        """the normed stream before the head, of the sequences' rows end to end"""
        H, K, D = self.heads, self.key_heads, self.D
        h = dropout(self.embed[tokens], P, seed, 0)
        y = rms_norm(h, self.norms[0])
        for i in range(len(self.W) // 4):
            qkv, out, into, back = self.W[4 * i:4 * i + 4]
            n1, n2, n3, n4 = self.norms[4 * i + 1:4 * i + 5]
            t = (y @ qkv.T).view(len(tokens), H + 2 * K, D)
            t = attention(t[:, :H], t[:, H:H + K], t[:, H + K:], causal=True, q_starts=starts, max_q=longest)
            y, h = block_norm(t.reshape(len(tokens), H * D) @ out.T, h, n1, n2, scale=SCALE, p=P, seed=seed, index=2 * i + 1)
            value, gate = (y @ into.T).chunk(2, 1)
            y, h = block_norm(value @ back.T, h, n3, n4, gate=gate, scale=SCALE, p=P, seed=seed, index=2 * i + 2)
        return y


def gradients(model, tokens, targets, starts, longest, seed):
    """the loss, with the gradients in the parameters' grad"""
    for p in model.parameters():
        p.grad = None
    y = model.hidden(tokens, starts, longest, seed)
    loss, dy, model.head.grad = linear_cross_entropy_grad(y, model.head, targets)
    y.backward(dy)
    return loss


def step(model, tokens, targets, starts, longest, seed, rate=0.02, max_norm=1.0):
    """one training step; the loss and the gradients' norm as tensors on the device"""
    loss = gradients(model, tokens, targets, starts, longest, seed)
    params = model.parameters()
    clipped = [torch.empty(p.shape, dtype=torch.float32, device=p.device) for p in params]
    norm = clip_grad_norm([p.grad for p in params], max_norm, out=clipped)
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


def texts(g, vocab, lengths, device="cuda"):
    """(tokens, targets, starts): texts whose next token follows from this one and the one before; the first has no target"""
    n = sum(lengths)
    tokens = torch.randint(0, vocab, (n,), generator=g, device=device)
    starts = torch.tensor([0, *lengths], device=device).cumsum(0).to(torch.int32)
    before = torch.cat([tokens[:1], tokens[:-1]])
    targets = (3 * tokens + before) % vocab
    targets[starts[:-1][starts[:-1] < n].long()] = -100
    return tokens, targets, starts


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--vocab", type=int, default=50)
    args = ap.parse_args()
    model = Model(vocab=args.vocab)
    g = torch.Generator(device="cuda").manual_seed(1)
    lengths = [300, 1, 77, 512, 158]
    for i in range(args.steps):
        tokens, targets, starts = texts(g, args.vocab, lengths)
        loss, norm = step(model, tokens, targets, starts, max(lengths), seed=i)
        if i % 10 == 0 or i == args.steps - 1:
            print(f"step {i}: loss {float(loss):.4f}, gradient norm {float(norm):.4f}", flush=True)


if __name__ == "__main__":
    main()
