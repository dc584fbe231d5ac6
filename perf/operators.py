"""The training operators beside orth(X), as cases that can be timed and compared.

A training step of a language model whose layers are kept orthonormal by orth() ends in the loss over the vocabulary,
passes root-mean-square norms on its way back, and clips the gradients by their global norm before the optimizer forms
X = V (U^T U) + u^T U from them. So the cases are

  ce        N, H, V, type, ignored, grads   cross entropy of softmax(x W^T) against N targets, without keeping the
                                            logits; with its gradients dx and dW, or (grads false) one loss per token
  rms       rows, D, type, residual, quant, backward
                                            root-mean-square norm of the residual stream after the addition; its
                                            output in the model's type or in 8-bit floats with one scale a row; or
                                            forward and backward together
  clip      kind, layers, type, out         the global norm over many tensors and the clipped copies of them (in 32
                                            bits where the optimizer works in 32 bits), or the norm alone

at the hidden and layer sizes of the models that spanqr_amd/qrbench/gen.py names (768 and 2048 wide for 110M, 1024 and
3584 for 0.8B, 5120, 6144 and 17408 for 27B) and at generic vocabularies.

Definitions: a token whose target is IGNORE has no loss and no gradient, and the mean is over the others. The stream
h = x + residual is rounded to its type once and the norm is of h as it is kept, so that forward and backward see the
same numbers. The 8-bit form is q = fp8(y 448 / max|y|) with scale max|y| / 448 a row, y in 32 bits.
"""
import math

import torch

own = False

IGNORE = -100
EPS = 1e-6
FP8_MAX = 448.0
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the log-probability of one token (a score in a search, or a single step of an evaluation): latency and one
        # read of the head's weights
        {"name": "ce_score_1", "op": "ce", "N": 1, "H": 1024, "V": 32000, "type": "bf16", "ignored": 0.0, "grads": False},
        # scoring a ragged batch of held-out text: no gradient, one loss a token
        {"name": "ce_score_1999", "op": "ce", "N": 1999, "H": 2048, "V": 50257, "type": "bf16", "ignored": 0.0,
         "grads": False},
        # training step of the 110M model, a small batch
        {"name": "ce_train_512", "op": "ce", "N": 512, "H": 768, "V": 32000, "type": "bf16", "ignored": 0.0, "grads": True},
        # the 0.8B model with padding in the batch; an odd vocabulary, and half precision
        {"name": "ce_train_4000", "op": "ce", "N": 4000, "H": 1024, "V": 50257, "type": "fp16", "ignored": 0.1,
         "grads": True},
        # the 27B model's head at a full batch
        {"name": "ce_train_8192", "op": "ce", "N": 8192, "H": 5120, "V": 128000, "type": "bf16", "ignored": 0.02,
         "grads": True},
        # one token on its way through a layer whose next product takes 8 bits: latency
        {"name": "rms_token", "op": "rms", "rows": 1, "D": 5120, "type": "bf16", "residual": True, "quant": True,
         "backward": False},
        # a prompt on the same way
        {"name": "rms_prompt", "op": "rms", "rows": 4096, "D": 5120, "type": "bf16", "residual": True, "quant": True,
         "backward": False},
        # training, forward and backward with the residual's gradient
        {"name": "rms_train", "op": "rms", "rows": 16384, "D": 2048, "type": "bf16", "residual": True, "quant": False,
         "backward": True},
        # odd sizes in 32 bits, no residual (the norm behind an embedding)
        {"name": "rms_odd", "op": "rms", "rows": 3001, "D": 769, "type": "fp32", "residual": False, "quant": False,
         "backward": True},
        # the layers of a 110M model: clipped copies for the optimizer
        {"name": "clip_110m", "op": "clip", "kind": "110m", "layers": 12, "type": "fp32", "out": "fp32"},
        # all layers of a 27B model at rank 256, 16-bit gradients into a 32-bit optimizer
        {"name": "clip_27b", "op": "clip", "kind": "27b", "layers": 64, "type": "bf16", "out": "fp32"},
        # the norm alone, as it is logged every step: many ragged tensors
        {"name": "norm_ragged", "op": "clip", "kind": "ragged", "layers": 100, "type": "bf16", "out": "none"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: every operator over its whole range, odd sizes among them."""
    op = rng.choice(["ce", "ce", "rms", "rms", "clip"])
    if op == "ce":
        grads = rng.random() < 0.6
        N = _log_int(rng, 1, 8192)
        H = rng.choice([_log_int(rng, 64, 5120), 8 * _log_int(rng, 8, 640), 256 * rng.randint(1, 20)])
        V = rng.choice([_log_int(rng, 1000, 128000), 64 * _log_int(rng, 16, 2000)])
        return {"op": "ce", "N": N, "H": H, "V": V, "type": rng.choice(["bf16", "bf16", "fp16"]),
                "ignored": rng.choice([0.0, 0.05, 0.5]), "grads": grads}
    if op == "rms":
        D = rng.choice([_log_int(rng, 32, 17408), 64 * _log_int(rng, 1, 272)])
        most = min(65536, (16384 * 5120) // D)
        backward = rng.random() < 0.5
        return {"op": "rms", "rows": _log_int(rng, 1, most), "D": D, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "residual": rng.random() < 0.7, "quant": not backward and rng.random() < 0.6, "backward": backward}
    kind = rng.choice(["110m", "0.8b", "27b", "ragged"])
    most = {"110m": 48, "0.8b": 64, "27b": 64, "ragged": 400}[kind]
    kept = rng.choice(["bf16", "fp16", "fp32"])
    return {"op": "clip", "kind": kind, "layers": _log_int(rng, 1, most), "type": kept,
            "out": rng.choice(["none", "fp32", kept])}


def _shapes(case):
    """the gradients' shapes: the factored layers at rank 256 or 512 with their norms' weights, or ragged tensors of one
    element to some hundred thousand"""
    n = case["layers"]
    layer = {"110m": [(768, 512), (2048, 512), (768,)], "0.8b": [(1024, 256), (2048, 256), (3584, 256), (1024,)],
             "27b": [(5120, 256), (6144, 256), (17408, 256), (5120,)]}
    if case["kind"] in layer:
        return layer[case["kind"]] * n
    return [(1 + (i * 7919) % 613, 1 + (i * 104729) % 1021) for i in range(n)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] == "ce":
        N, H, V = case["N"], case["H"], case["V"]
        # logits of standard deviation 2.5; the target's own is 12 above the others' mean, as after some training
        W = (normal(V, H) * (2.5 / math.sqrt(H))).to(t)
        target = torch.randint(0, V, (N,), generator=g, device="cuda")
        s["x"] = (normal(N, H) + (12.0 / 6.25) * W[target].float()).to(t)
        s["W"] = W
        drop = torch.rand(N, generator=g, device="cuda") < case["ignored"]
        drop[0] = False
        s["target"] = torch.where(drop, torch.full_like(target, IGNORE), target)
    elif case["op"] == "rms":
        shape = (case["rows"], case["D"])
        # a stream whose rows differ in size and that has a few large channels
        wide = 1.0 + 9.0 * (torch.rand(case["D"], generator=g, device="cuda") < 0.01).float()
        s["x"] = (normal(*shape) * wide * torch.exp(0.5 * normal(case["rows"], 1))).to(t)
        s["residual"] = (normal(*shape) * wide).to(t) if case["residual"] else None
        s["weight"] = (1.0 + 0.1 * normal(case["D"])).to(t)
        if case["backward"]:
            s["dy"] = normal(*shape).to(t)
            s["dh"] = normal(*shape).to(t) if case["residual"] else None
    else:
        shapes = _shapes(case)
        total = sum(math.prod(x) for x in shapes)
        s["flat"] = (normal(total) * 0.01).to(t)   # one bucket, the tensors lie in it end to end
        s["grads"] = _views(s["flat"], shapes)
        s["max_norm"] = 0.5 * 0.01 * math.sqrt(total)
        if case["out"] != "none":
            s["out"] = torch.empty(total, device="cuda", dtype=TYPES[case["out"]])
            s["outs"] = _views(s["out"], shapes)
    return s


def _views(flat, shapes):
    sizes = [math.prod(x) for x in shapes]
    return [v.view(x) for v, x in zip(torch.split(flat, sizes), shapes)]


def _ce(x, W, target, grads):
    """the loss of each token (grads false), or the mean loss with dx and dW"""
    xf, Wf = x.float(), W.float()
    z = xf @ Wf.T
    m = z.amax(1, keepdim=True)
    kept = target != IGNORE
    at = torch.where(kept, target, torch.zeros_like(target))[:, None]
    zt = z.gather(1, at)
    e = z.sub_(m).exp_()
    total = e.sum(1, keepdim=True)
    loss = torch.where(kept, (m + total.log() - zt)[:, 0], torch.zeros_like(m[:, 0]))
    if not grads:
        return loss
    n = kept.sum().float()
    p = e.div_(total)
    p.scatter_add_(1, at, torch.full_like(zt, -1.0))
    p.mul_(kept[:, None].float() / n)
    return loss.sum() / n, (p @ Wf).to(x.dtype), (p.T @ xf).to(W.dtype)


def _rms(s):
    x, w = s["x"], s["weight"]
    h = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    hf, wf = h.float(), w.float()
    rstd = torch.rsqrt((hf * hf).mean(1, keepdim=True) + EPS)
    n = hf * rstd
    y = n * wf
    out = {} if s["residual"] is None else {"h": h}
    if s["case"]["quant"]:
        amax = y.abs().amax(1, keepdim=True)
        out["q"] = (y * (FP8_MAX / amax)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
        out["scale"] = (amax / FP8_MAX)[:, 0]
    else:
        out["y"] = y.to(x.dtype)
    if s["case"]["backward"]:
        dy = s["dy"].float()
        dn = dy * wf
        dx = rstd * (dn - n * (dn * n).mean(1, keepdim=True))
        out["dx"] = (dx if s["dh"] is None else dx + s["dh"].float()).to(x.dtype)
        out["dw"] = (dy * n).sum(0).to(w.dtype)
    return out


def _clip(s):
    total = torch.stack([v.float().square().sum() for v in s["grads"]]).sum()
    norm = total.sqrt()
    if s["case"]["out"] == "none":
        return norm
    scale = torch.clamp(s["max_norm"] / norm, max=1.0)
    [o.copy_(v.float() * scale) for o, v in zip(s["outs"], s["grads"])]
    return norm, s["out"]


def run(s):
    case = s["case"]
    if not own:
        if case["op"] == "ce":
            return _ce(s["x"], s["W"], s["target"], case["grads"])
        return _rms(s) if case["op"] == "rms" else _clip(s)
    import spanqr_amd as sp
    if case["op"] == "ce":
        if case["grads"]:
            return sp.linear_cross_entropy_grad(s["x"], s["W"], s["target"], ignore_index=IGNORE)
        return sp.linear_cross_entropy(s["x"], s["W"], s["target"], ignore_index=IGNORE, reduction="none")
    if case["op"] == "rms":
        out = {}
        got = sp.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, quant="fp8" if case["quant"] else None)
        got = got if isinstance(got, tuple) else (got,)
        if case["quant"]:
            out["q"], out["scale"] = got[:2]
        else:
            out["y"] = got[0]
        h = s["x"]
        if s["residual"] is not None:
            h = out["h"] = got[-1]
        if case["backward"]:
            out["dx"], out["dw"] = sp.rms_norm_backward(s["dy"], h, s["weight"], eps=EPS, dh=s["dh"])
        return out
    if case["out"] == "none":
        return sp.grad_norm(s["grads"])
    return sp.clip_grad_norm(s["grads"], s["max_norm"], out=s["outs"]), s["out"]


def work(case):
    if case["op"] == "ce":
        N, H, V, b = case["N"], case["H"], case["V"], BYTES[case["type"]]
        read = b * (N * H + V * H) + 8 * N
        if case["grads"]:
            return {"bytes": 2 * b * (N * H + V * H) + 8 * N + 4, "flops": 6 * N * H * V}
        return {"bytes": read + 4 * N, "flops": 2 * N * H * V}
    if case["op"] == "rms":
        n, D, b = case["rows"] * case["D"], case["D"], BYTES[case["type"]]
        moved = n * b + D * b                                         # x, weight
        moved += 2 * n * b if case["residual"] else 0                 # residual, h
        moved += n + 4 * case["rows"] if case["quant"] else n * b     # q and scale, or y
        if case["backward"]:
            moved += 3 * n * b + 2 * D * b                            # dy, h again, dx; weight again, dw
            moved += n * b if case["residual"] else 0                 # the stream's own gradient
        return {"bytes": moved, "flops": (12 if case["backward"] else 4) * n}
    total = sum(math.prod(x) for x in _shapes(case))
    out = 0 if case["out"] == "none" else BYTES[case["out"]]
    return {"bytes": total * (BYTES[case["type"]] + out) + 4, "flops": (3 if out else 2) * total}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ce":
        return _exact_ce(s, case)
    if case["op"] == "rms":
        return _exact_rms(s, case)
    v = s["flat"].double()
    norm = torch.linalg.vector_norm(v)
    if case["out"] == "none":
        return norm
    return norm, v * min(1.0, s["max_norm"] / norm.item())


def _exact_ce(s, case):
    """in pieces of the tokens, from log softmax and the one-hot matrix"""
    x, W, target = s["x"].double(), s["W"].double(), s["target"]
    n = int((target != IGNORE).sum())
    losses, dxs, dW = [], [], torch.zeros_like(W) if case["grads"] else None
    for i in range(0, case["N"], 2048):
        xi, ti = x[i:i + 2048], target[i:i + 2048]
        rows = torch.nonzero(ti != IGNORE)[:, 0]
        logp = torch.log_softmax(xi @ W.T, dim=1)
        loss = torch.zeros(len(ti), device=x.device, dtype=torch.float64)
        loss[rows] = -logp[rows, ti[rows]]
        losses.append(loss)
        if case["grads"]:
            G = torch.zeros_like(logp)
            G[rows] = logp[rows].exp()
            G[rows, ti[rows]] -= 1.0
            G /= n
            dxs.append(G @ W)
            dW += G.T @ xi
    if case["grads"]:
        return torch.cat(losses).sum() / n, torch.cat(dxs), dW
    return torch.cat(losses)


def _exact_rms(s, case):
    D = case["D"]
    h = s["x"] if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(s["x"].dtype)
    H, w = h.double(), s["weight"].double()
    root = torch.sqrt(torch.linalg.vector_norm(H, dim=1, keepdim=True) ** 2 / D + EPS)
    out = {} if s["residual"] is None else {"h": h.double()}
    y = H / root * w
    if case["quant"]:
        scale = torch.linalg.vector_norm(y, ord=math.inf, dim=1) / FP8_MAX
        q = (y / scale[:, None]).clamp(-FP8_MAX, FP8_MAX)
        out["q"], out["scale"] = q.float().to(torch.float8_e4m3fn).double(), scale
    else:
        out["y"] = y
    if case["backward"]:
        dy = s["dy"].double()
        c = torch.einsum("rd,rd->r", dy * w, H)[:, None] / (D * root ** 3)
        dx = dy * w / root - H * c
        out["dx"] = dx if s["dh"] is None else dx + s["dh"].double()
        out["dw"] = torch.einsum("rd,rd->d", dy, H / root)
    return out
