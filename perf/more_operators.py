"""The operators between the embedding and the loss of a training step, as cases that can be timed and compared.

A block of a language model mixes its tokens with attention and hands the result on through norms: one behind the block,
scaled by a gate, thinned by dropout and added to the residual stream, and one in front of the next block. So the
cases are

  attn   B, Sq, Sk, heads, kv_heads, D, type, causal, window, packed, backward
                                        softmax attention with heads that share keys and values; forward alone (one
                                        token against what is cached, or a prompt), or forward and backward together;
                                        as a batch [B, S, heads, D], or packed as sequences of ragged lengths end to end
  join   rows, D, type, gate, p, backward
                                        t = norm(x) w1 silu(gate), h = residual + scale dropout(t), y = norm(h) w2;
                                        forward, or forward and backward together
  drop   rows, D, type, p               dropout of x, and of the gradient that comes back through it

at the widths of the models that spanqr_amd/qrbench/gen.py names (768 wide for 110M, 1024 for 0.8B, 5120 for 27B), in
heads of 64 and 128, and at generic lengths.

Definitions. Attention: query i of a sequence of Lq queries and Lk keys stands at p = i + Lk - Lq; causal: it sees the keys
j <= p, with a window w only those with j > p - w too. A query that sees no key has output 0. The stream h is rounded to its
type once and normed as rounded. Dropout: element (row, column) is dropped where its 16-bit number is below P =
round(65536 p), the others are multiplied by 65536 / (65536 - P). Its number is half (column % 2) of word
(column % 8) / 2 (low half first) of Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as
1, 2, 3; 2011) with counter (column / 8, row mod 2^32, row / 2^32, index) and the seed's low and high words as key.
"""
import math
import random

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
SCALE = 0.5          # of what a block adds to the stream
INDEX = 3            # which dropout of the step this is


def _attn(name, B, Sq, Sk, heads, kv_heads, D, type="bf16", causal=True, window=0, packed=False, backward=True):
    c = {"op": "attn", "B": B, "Sq": Sq, "Sk": Sk, "heads": heads, "kv_heads": kv_heads, "D": D, "type": type,
         "causal": causal, "window": window, "packed": packed, "backward": backward}
    return dict({"name": name}, **c) if name else c


def listed():
    return [
        # one token of the 27B model against a long context: latency, and one read of its keys and values
        _attn("attn_token", 1, 1, 8191, 40, 8, 128, backward=False),
        # one token each for 32 requests whose contexts are of ragged lengths, end to end in memory
        _attn("attn_tokens_32", 32, 1, 4096, 16, 2, 128, "fp16", packed=True, backward=False),
        # the smallest training step: a few short texts
        _attn("attn_train_small", 2, 100, 100, 12, 12, 64),
        # a training step of the 110M model
        _attn("attn_train_1024", 16, 1024, 1024, 12, 12, 64),
        # a training batch of the 0.8B model packed from texts of ragged lengths, with a window, in half precision
        _attn("attn_train_ragged", 24, 2048, 2048, 8, 2, 128, "fp16", window=1000, packed=True),
        # one long text in training at the 27B model's width
        _attn("attn_train_16384", 1, 16384, 16384, 40, 8, 128),
        # an encoder's batch: every token sees every other, an odd length and an unusual head
        _attn("attn_encode_1999", 4, 1999, 1999, 16, 16, 80, causal=False, backward=False),
        # one token on its way from a block to the next: latency
        {"name": "join_token", "op": "join", "rows": 1, "D": 5120, "type": "bf16", "gate": True, "p": 0.0, "backward": False},
        # training with everything on
        {"name": "join_train", "op": "join", "rows": 16384, "D": 2048, "type": "bf16", "gate": True, "p": 0.1, "backward": True},
        # odd sizes in 32 bits, without gate and dropout
        {"name": "join_odd", "op": "join", "rows": 3001, "D": 769, "type": "fp32", "gate": False, "p": 0.0, "backward": True},
        # a small batch behind the embedding of the 110M model
        {"name": "drop_small", "op": "drop", "rows": 512, "D": 768, "type": "fp32", "p": 0.1},
        # the stream of the 27B model
        {"name": "drop_large", "op": "drop", "rows": 16384, "D": 5120, "type": "bf16", "p": 0.05},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: every operator over its whole range, odd sizes among them."""
    op = rng.choice(["attn", "attn", "attn", "join", "join", "drop"])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if op == "attn":
        group, kv_heads = rng.choice([1, 1, 2, 3, 4, 5, 8]), rng.choice([1, 2, 3, 4, 8, 12])
        D = rng.choice([64, 128, 64, 128, 8 * rng.randint(1, 16)])
        packed = rng.random() < 0.4
        if rng.random() < 0.3:   # a few tokens against a cache
            B, Sq, Sk = _log_int(rng, 1, 64), rng.choice([1, 1, 1, _log_int(rng, 2, 16)]), _log_int(rng, 16, 32768)
            while B * Sk > 1 << 18:
                B = max(1, B // 2)
            return _attn(None, B, Sq, Sk, group * kv_heads, kv_heads, D, kind, packed=packed, backward=False)
        Sq = _log_int(rng, 16, 8192)
        B = _log_int(rng, 1, 32)
        while B * group * kv_heads * Sq * Sq > 1 << 31:
            B, Sq = max(1, B // 2), Sq if B > 1 else Sq // 2
        Sk = Sq if rng.random() < 0.8 else _log_int(rng, 16, 2 * Sq)
        causal = rng.random() < 0.7
        window = _log_int(rng, 16, Sq) if causal and rng.random() < 0.3 else 0
        return _attn(None, B, Sq, Sk, group * kv_heads, kv_heads, D, kind, causal, window, packed, rng.random() < 0.7)
    D = rng.choice([_log_int(rng, 32, 17408), 64 * _log_int(rng, 1, 272)])
    most = min(65536, (16384 * 5120) // D)
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "join":
        return {"op": "join", "rows": _log_int(rng, 1, most), "D": D, "type": kind, "gate": rng.random() < 0.6,
                "p": rng.choice([0.0, 0.1, 0.25]), "backward": rng.random() < 0.6}
    return {"op": "drop", "rows": _log_int(rng, 1, most), "D": D, "type": kind, "p": rng.choice([0.05, 0.1, 0.5])}


def _lengths(case):
    """(queries, keys) of each sequence. Packed: ragged ones, an empty one and one of a single token among them where
    there are enough; one token each stays one."""
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    if not case["packed"]:
        return [(Sq, Sk)] * B
    rng = random.Random(1000 * B + Sq + Sk)
    out = []
    for b in range(B):
        part = 1.0 if b == 0 else rng.uniform(0.02, 1.0)
        k = 0 if b == 5 else 1 if b == 6 else max(1, int(part * Sk))
        out.append((min(Sq, k) if Sq < 32 else (k if Sq == Sk else max(1, int(part * Sq))), k))
    return out


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] == "attn":
        H, Hk, D = case["heads"], case["kv_heads"], case["D"]
        lengths = _lengths(case)
        s["lengths"] = lengths
        if case["packed"]:
            qs, ks = _starts([q for q, _ in lengths]), _starts([k for _, k in lengths])
            s["q_starts"] = torch.tensor(qs, dtype=torch.int32, device="cuda")
            s["k_starts"] = torch.tensor(ks, dtype=torch.int32, device="cuda")
            s["max_q"], s["max_k"] = max(q for q, _ in lengths), max(k for _, k in lengths)
            q_shape, k_shape = (qs[-1],), (ks[-1],)
        else:
            q_shape, k_shape = (case["B"], case["Sq"]), (case["B"], case["Sk"])
        if q_shape == k_shape:
            # one product gives all three; queries, keys and values are its columns
            qkv = normal(*q_shape, H + 2 * Hk, D)
            qkv[..., :H + Hk, :] *= 1.5
            qkv = qkv.to(t)
            s["q"], s["k"], s["v"] = qkv[..., :H, :], qkv[..., H:H + Hk, :], qkv[..., H + Hk:, :]
        else:
            s["q"] = (1.5 * normal(*q_shape, H, D)).to(t)
            s["k"] = (1.5 * normal(*k_shape, Hk, D)).to(t)
            s["v"] = normal(*k_shape, Hk, D).to(t)
        if case["backward"]:
            s["dout"] = normal(*q_shape, H, D).to(t)
        return s
    shape = (case["rows"], case["D"])
    s["x"] = normal(*shape)
    if case["op"] == "drop":
        s["x"], s["dy"] = s["x"].to(t), normal(*shape).to(t)
    else:
        # a block's output and a stream whose rows differ in size and that has a few large channels
        wide = 1.0 + 9.0 * (torch.rand(case["D"], generator=g, device="cuda") < 0.01).float()
        s["x"] = (s["x"] * torch.exp(0.5 * normal(case["rows"], 1))).to(t)
        s["residual"] = (normal(*shape) * wide).to(t)
        s["gate"] = normal(*shape).to(t) if case["gate"] else None
        s["post_weight"], s["weight"] = ((1.0 + 0.1 * normal(case["D"])).to(t) for _ in range(2))
        if case["backward"]:
            s["dy"], s["dh"] = normal(*shape).to(t), normal(*shape).to(t)
    # the step's own seed, on the device: a captured step takes another one in each replay
    s["seed"] = torch.randint(-1 << 62, 1 << 62, (1,), generator=g, device="cuda", dtype=torch.int64)
    return s


def _seen(lq, lk, case, device):
    """[lq, lk]: which keys a query sees"""
    j = torch.arange(lk, device=device)[None, :]
    p = torch.arange(lq, device=device)[:, None] + (lk - lq)
    seen = torch.ones(lq, lk, dtype=torch.bool, device=device)
    if case["causal"]:
        seen = j <= p
        if case["window"]:
            seen = seen & (j > p - case["window"])
    return seen


def _attention(q, k, v, dout, seen, scale, out, grads):
    """of a few heads: q [n, Lq, D], k and v [n / group, Lk, D] in the model's type, into out [n, Lq, D] and grads"""
    group = q.shape[0] // k.shape[0]
    qf = q.float()
    kf, vf = (x.float().repeat_interleave(group, 0) for x in (k, v))
    s = (qf @ kf.transpose(1, 2)).mul_(scale).masked_fill_(~seen, -math.inf)
    m = s.amax(2, keepdim=True) if s.shape[2] else s.new_zeros(s.shape[0], s.shape[1], 1)
    p = s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = p.sum(2, keepdim=True)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    out.copy_(p @ vf)
    if dout is None:
        return
    dq, dk, dv = grads
    df = dout.float()
    dv.copy_((p.transpose(1, 2) @ df).view(v.shape[0], group, *v.shape[1:]).sum(1))
    dp = df @ vf.transpose(1, 2)
    ds = p.mul_(dp.sub_((p * dp).sum(2, keepdim=True))).mul_(scale)
    dq.copy_(ds @ kf)
    dk.copy_((ds.transpose(1, 2) @ qf).view(k.shape[0], group, *k.shape[1:]).sum(1))


def _attn_plain(s):
    case = s["case"]
    q, k, v, dout = s["q"], s["k"], s["v"], s.get("dout")
    group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["D"])
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    grads = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v)] if dout is not None else None
    if case["packed"]:
        sequences = []
        qa = ka = 0
        for lq, lk in s["lengths"]:
            sequences.append((slice(qa, qa + lq), slice(ka, ka + lk), lq, lk))
            qa, ka = qa + lq, ka + lk
    else:
        sequences = [(b, b, case["Sq"], case["Sk"]) for b in range(case["B"])]
    seen = None
    for qa, ka, lq, lk in sequences:
        if seen is None or seen.shape != (lq, lk):
            seen = _seen(lq, lk, case, q.device)
        # as many heads at once as keep a matrix of scores below 2 GiB
        step = max(1, min(case["kv_heads"], (1 << 29) // max(1, group * lq * lk)))
        for h in range(0, case["kv_heads"], step):
            hk, hq = slice(h, h + step), slice(h * group, (h + step) * group)

            def at(x, a, hs):
                return x[a][:, hs].transpose(0, 1)
            _attention(at(q, qa, hq), at(k, ka, hk), at(v, ka, hk), None if dout is None else at(dout, qa, hq), seen, scale,
                       at(out, qa, hq), None if grads is None else
                       (at(grads[0], qa, hq), at(grads[1], ka, hk), at(grads[2], ka, hk)))
    return {"out": out} if dout is None else {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}


def _kept(rows, D, p, seed):
    """[rows, D]: which elements dropout keeps"""
    low = 0xFFFFFFFF
    c = [torch.arange((D + 7) // 8, device=seed.device)[None, :], torch.arange(rows, device=seed.device)[:, None],
         torch.zeros((1, 1), dtype=torch.int64, device=seed.device), torch.full((1, 1), INDEX, device=seed.device)]
    key = [seed & low, (seed >> 32) & low]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57   # (modulo 2^64)
        c = [((b >> 32) & low) ^ c[1] ^ key[0], b & low, ((a >> 32) & low) ^ c[3] ^ key[1], a & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    words = torch.stack(torch.broadcast_tensors(*c), 2)
    number = torch.stack([words & 0xFFFF, words >> 16], 3).reshape(rows, -1)[:, :D]
    return number >= round(65536 * p)


def _factor(p):
    return 65536 / (65536 - round(65536 * p))


def _join_plain(s):
    case = s["case"]
    x, r = s["x"], s["residual"]
    w1, w2 = s["post_weight"].float(), s["weight"].float()
    xf = x.float()
    s1 = torch.rsqrt((xf * xf).mean(1, keepdim=True) + EPS)
    n1 = xf * s1
    t = n1 * w1
    if case["gate"]:
        g = s["gate"].float()
        sig = 1.0 / (1.0 + torch.exp(-g))
        t = t * (g * sig)
    f = SCALE
    if case["p"] > 0.0:
        f = torch.where(_kept(*x.shape, case["p"], s["seed"]), SCALE * _factor(case["p"]), 0.0)
    h = (r.float() + t * f).to(x.dtype)
    hf = h.float()
    s2 = torch.rsqrt((hf * hf).mean(1, keepdim=True) + EPS)
    n2 = hf * s2
    out = {"y": (n2 * w2).to(x.dtype), "h": h}
    if case["backward"]:
        dy = s["dy"].float()
        u2 = dy * w2
        dr = s2 * (u2 - n2 * (u2 * n2).mean(1, keepdim=True)) + s["dh"].float()
        dt = dr * f
        out["dresidual"], out["dweight"] = dr.to(x.dtype), (dy * n2).sum(0).to(x.dtype)
        if case["gate"]:
            out["dgate"] = (dt * n1 * w1 * (sig * (1.0 + g * (1.0 - sig)))).to(x.dtype)
            dt = dt * (g * sig)
        u1 = dt * w1
        out["dx"] = (s1 * (u1 - n1 * (u1 * n1).mean(1, keepdim=True))).to(x.dtype)
        out["dpost_weight"] = (dt * n1).sum(0).to(x.dtype)
    return out


def run(s):
    case = s["case"]
    if not own:
        if case["op"] == "attn":
            return _attn_plain(s)
        if case["op"] == "join":
            return _join_plain(s)
        f = torch.where(_kept(case["rows"], case["D"], case["p"], s["seed"]), _factor(case["p"]), 0.0)
        return {"y": (s["x"].float() * f).to(s["x"].dtype), "dx": (s["dy"].float() * f).to(s["x"].dtype)}
    import spanqr_amd as sp
    if case["op"] == "attn":
        how = {"causal": case["causal"], "window": case["window"] or None}
        if case["packed"]:
            how.update(q_starts=s["q_starts"], k_starts=s["k_starts"], max_q=s["max_q"], max_k=s["max_k"])
        if not case["backward"]:
            return {"out": sp.attention(s["q"], s["k"], s["v"], **how)}
        out, lse = sp.attention(s["q"], s["k"], s["v"], return_lse=True, **how)
        dq, dk, dv = sp.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **how)
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if case["op"] == "drop":
        return {"y": sp.dropout(s["x"], case["p"], s["seed"], INDEX), "dx": sp.dropout(s["dy"], case["p"], s["seed"], INDEX)}
    how = {"gate": s["gate"], "scale": SCALE, "p": case["p"], "seed": s["seed"], "index": INDEX, "eps": EPS}
    y, h = sp.block_norm(s["x"], s["residual"], s["post_weight"], s["weight"], **how)
    out = {"y": y, "h": h}
    if case["backward"]:
        g = sp.block_norm_backward(s["dy"], s["dh"], s["x"], h, s["post_weight"], s["weight"], **how)
        out.update(dresidual=g.residual, dweight=g.weight, dx=g.x, dpost_weight=g.post_weight)
        if case["gate"]:
            out["dgate"] = g.gate
    return out


def _pairs(lq, lk, case):
    """how many (query, key) pairs count"""
    if not case["causal"]:
        return lq * lk
    total, w = 0, case["window"] or lk + lq
    for i in range(lq):
        p = i + lk - lq
        if p >= 0:
            total += min(p + 1, lk) - max(0, p - w + 1)
    return total


def work(case):
    b = BYTES[case["type"]]
    if case["op"] == "attn":
        lengths, D = _lengths(case), case["D"]
        n_q = sum(q for q, _ in lengths) * case["heads"] * D * b
        n_k = sum(k for _, k in lengths) * case["kv_heads"] * D * b
        pairs = sum(_pairs(*n, case) for n in set(lengths)) if len(set(lengths)) == len(lengths) else sum(
            _pairs(*n, case) * lengths.count(n) for n in set(lengths))
        forward = 2 * n_q + 2 * n_k                 # q, out; k, v
        if not case["backward"]:
            return {"bytes": forward, "flops": 4 * pairs * case["heads"] * D}
        # again q, out, k, v; dout, dq, dk, dv
        return {"bytes": forward + 4 * n_q + 4 * n_k, "flops": 14 * pairs * case["heads"] * D}
    n = case["rows"] * case["D"]
    if case["op"] == "drop":
        return {"bytes": 4 * n * b, "flops": 2 * n}
    moved = (5 if case["gate"] else 4) * n          # x, residual, gate; h, y
    if case["backward"]:
        moved += (8 if case["gate"] else 6) * n     # dy, dh, x, h, gate; dresidual, dx, dgate
    return {"bytes": moved * b + (6 if case["backward"] else 2) * case["D"] * b, "flops": (45 if case["backward"] else 15) * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attn(s, case)
    keep = _exact_kept(s, case) if case["p"] > 0.0 else None
    if case["op"] == "drop":
        part = 1.0 - round(65536 * case["p"]) / 65536
        zero = torch.zeros((), dtype=torch.float64, device="cuda")
        return {n: torch.where(keep, s[k].double() / part, zero) for n, k in (("y", "x"), ("dx", "dy"))}
    return _exact_join(s, case, keep)


def _exact_attn(s, case):
    """head by head of the queries, from the normalised probabilities and the softmax's Jacobian"""
    group, scale = case["heads"] // case["kv_heads"], case["D"] ** -0.5
    q, k, v = s["q"], s["k"], s["v"]
    if not case["packed"]:
        q, k, v = q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1)
    out = {"out": torch.zeros(q.shape, dtype=torch.float64, device="cuda")}
    dout = None
    if case["backward"]:
        dout = s["dout"] if case["packed"] else s["dout"].flatten(0, 1)
        out.update({n: torch.zeros(x.shape, dtype=torch.float64, device="cuda") for n, x in (("dq", q), ("dk", k), ("dv", v))})
    q0 = k0 = 0
    for lq, lk in s["lengths"]:
        q1, k1 = q0 + lq, k0 + lk
        if lq and lk:
            at = torch.arange(lk - lq, lk, device="cuda")
            far = at[:, None] - torch.arange(lk, device="cuda")[None, :]      # how far behind the query a key is
            hidden = (far < 0) if case["causal"] else torch.zeros_like(far, dtype=torch.bool)
            if case["window"]:
                hidden |= far >= case["window"]
            empty = hidden.all(1)
            for h in range(case["heads"]):
                Q, K, V = q[q0:q1, h].double(), k[k0:k1, h // group].double(), v[k0:k1, h // group].double()
                z = torch.where(hidden, torch.full_like(far, -math.inf, dtype=torch.float64), scale * (Q @ K.T))
                P = torch.softmax(z, 1)
                P[empty] = 0.0
                out["out"][q0:q1, h] = P @ V
                if dout is not None:
                    G = dout[q0:q1, h].double()
                    gP = G @ V.T
                    dz = P * gP
                    dz -= P * torch.einsum("ij,ij->i", P, gP)[:, None]
                    out["dq"][q0:q1, h] = scale * (dz @ K)
                    out["dk"][k0:k1, h // group] += scale * (dz.T @ Q)
                    out["dv"][k0:k1, h // group] += P.T @ G
        q0, k0 = q1, k1
    if not case["packed"]:
        for n, like in (("out", s["q"]), ("dq", s["q"]), ("dk", s["k"]), ("dv", s["v"])):
            if n in out:
                out[n] = out[n].view(like.shape)
    return out


def _exact_kept(s, case):
    """the generator in 16-bit limbs, row by row of counters"""
    rows, blocks = case["rows"], -(-case["D"] // 8)

    def times(m, c):
        """high and low 32 bits of m c"""
        m1, m0, c1, c0 = m >> 16, m & 0xFFFF, torch.div(c, 65536, rounding_mode="floor"), c % 65536
        mid = m1 * c0 + torch.div(m0 * c0, 65536, rounding_mode="floor")
        mid2 = m0 * c1 + mid % 65536
        return m1 * c1 + torch.div(mid, 65536, rounding_mode="floor") + torch.div(mid2, 65536, rounding_mode="floor"), \
            (mid2 % 65536) * 65536 + (m0 * c0) % 65536
    seed = int(s["seed"]) % 2 ** 64
    k0, k1 = seed % 2 ** 32, seed // 2 ** 32
    n = torch.arange(rows * blocks, device="cuda")
    x0, x1 = n % blocks, torch.div(n, blocks, rounding_mode="floor")
    x2, x3 = torch.zeros_like(n), torch.full_like(n, INDEX)
    for r in range(10):
        h0, l0 = times(0xD2511F53, x0)
        h1, l1 = times(0xCD9E8D57, x2)
        x0, x1, x2, x3 = h1 ^ x1 ^ ((k0 + r * 0x9E3779B9) % 2 ** 32), l1, h0 ^ x3 ^ ((k1 + r * 0xBB67AE85) % 2 ** 32), l0
    halves = [f(x) for x in (x0, x1, x2, x3) for f in (lambda x: x % 65536, lambda x: torch.div(x, 65536, rounding_mode="floor"))]
    u = torch.stack([h.view(rows, blocks) for h in halves], 2).view(rows, 8 * blocks)[:, :case["D"]]
    return ~(u < round(case["p"] * 65536))


def _exact_join(s, case, keep):
    D = case["D"]
    x, w1, w2 = s["x"].double(), s["post_weight"].double(), s["weight"].double()
    root1 = torch.sqrt(torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / D + EPS)
    gate = torch.ones_like(x)
    if case["gate"]:
        gate = torch.nn.functional.silu(s["gate"].double())
    through = torch.full_like(x, SCALE)
    if keep is not None:
        through = through * keep / (1.0 - round(65536 * case["p"]) / 65536)
    h = (s["residual"].double() + through * gate * w1 * x / root1).to(s["x"].dtype)
    H = h.double()
    root2 = torch.sqrt(torch.linalg.vector_norm(H, dim=1, keepdim=True) ** 2 / D + EPS)
    # (y and the gradients are of the stream as it is rounded: where another rounding of h is as good, so are its own)
    out = {"y": H / root2 * w2, "h": h.double()}
    if case["backward"]:
        dy = s["dy"].double()
        c2 = torch.einsum("rd,rd->r", dy * w2, H)[:, None] / (D * root2 ** 3)
        dr = dy * w2 / root2 - H * c2 + s["dh"].double()
        dt = dr * through
        out["dresidual"], out["dweight"] = dr, torch.einsum("rd,rd->d", dy, H / root2)
        if case["gate"]:
            z = s["gate"].double()
            slope = torch.sigmoid(z) + torch.nn.functional.silu(z) * torch.sigmoid(-z)
            out["dgate"] = dt * slope * w1 * x / root1
        u = dt * gate * w1
        c1 = torch.einsum("rd,rd->r", u, x)[:, None] / (D * root1 ** 3)
        out["dx"] = u / root1 - x * c1
        out["dpost_weight"] = torch.einsum("rd,rd->d", dt * gate, x / root1)
    return out
