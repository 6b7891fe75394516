"""Measured cases of the packed-batch operators: the 8-bit integer linear layer, the per-head norm with
multi-axis rotation, and attention over packed sequences of different lengths.

A case is one pass through one operator.  `run` computes it either in plain form (elementary torch
operations in 32 bits, rounded once at the end) or, with `own` set, through the engine's entry points
in chroma-radiance_b200/b2g.py.  `exact` states each operator's definition in 64 bits.

    linear_s8         y = act((sum_k xq[m, k] wq[n, k]) xs[m] ws[n] + bias[n]) with 8-bit integers: per-token
                      xs[m] = max_k |x[m, k]| / 127, xq = round(x 127 / max), ties to even; per-channel
                      weights quantised when they were loaded
    qk_norm_rope      per head: x rsqrt(mean(x^2) + eps) w, then pair p turned by the angle
                      position[axis] theta^(-2 j / d_axis), the j-th pair of its axis
    attention_packed  softmax(q k^T scale) v within each sequence, a key head shared by a group of
                      query heads, optionally causal (the last query sees the last key)
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "s8": 1}
EPS = 1e-6
#: what one pass may cost at most: the largest listed case of each operator
MOST_MACS = 4608 * 21504 * 3072
MOST_VALUES = 29120 * 32 * 128
MOST_SCORES = 1.3e9      # query heads x padded queries x padded keys of all sequences
MOST_CACHE = 48 * 8192   # padded keys of all sequences


# ---------------------------------------------------------------------------- cases

def listed():
    return [
        # One token through a 5120-wide layer (the approximator's width): latency, the weight is all there is to read.
        dict(name="linear_s8 one token 5120x5120", op="linear_s8", m=1, n=5120, k=5120, x="bf16", out="bf16",
             act="none", bias=True),
        # The approximator's 344 modulation rows with its SiLU.
        dict(name="linear_s8 344 rows 5120x5120 silu", op="linear_s8", m=344, n=5120, k=5120, x="bf16", out="bf16",
             act="silu", bias=True),
        # The text encoder's feed-forward over the packed tokens of a few prompts (odd row count, fp16, GELU).
        dict(name="linear_s8 509 prompt tokens 4096 to 10240 gelu", op="linear_s8", m=509, n=10240, k=4096, x="f16",
             out="f16", act="gelu", bias=False),
        # The qkv projection at 512^2 of activations that another layer has quantised already; F32 result.
        dict(name="linear_s8 qkv of 1536 quantised tokens", op="linear_s8", m=1536, n=9216, k=3072, x="s8", out="f32",
             act="none", bias=True),
        # The single block's first layer at 1024^2.
        dict(name="linear_s8 4608 tokens 3072 to 21504 gelu", op="linear_s8", m=4608, n=21504, k=3072, x="bf16",
             out="bf16", act="gelu", bias=True),
        # One new token for each of 64 sequences, one position axis, halves rotated, grouped heads.
        dict(name="qk_norm_rope 64 single tokens", op="qk_norm_rope", t=64, hq=32, hk=8, d=128, axes="128",
             pairs="halves", x="bf16", out="bf16", norm=True, top=8000),
        # A 512^2 image with its 512 text tokens: 24 heads, axes 16/56/56, q and k read from the fused projection.
        dict(name="qk_norm_rope 1536 tokens 24 heads", op="qk_norm_rope", t=1536, hq=24, hk=24, d=128, axes="16,56,56",
             pairs="neighbours", x="bf16", out="bf16", norm=True, top=64),
        # A clip of 13 frames of 40 x 56 patches, F32 projection, grouped heads.
        dict(name="qk_norm_rope 29120 video tokens", op="qk_norm_rope", t=29120, hq=24, hk=8, d=128, axes="32,48,48",
             pairs="neighbours", x="f32", out="bf16", norm=True, top=64),
        # One query token for each of 48 caches of uneven fill.
        dict(name="attention_packed 48 single queries", op="attention_packed", mode="cache", b=48, low=1, high=8191,
             hq=32, hk=8, d=128, x="bf16", causal=True, shape=7),
        # A causal text model over a batch of prompts from a word to a long page.
        dict(name="attention_packed 40 causal prompts", op="attention_packed", mode="self", b=40, low=1, high=2047,
             hq=32, hk=8, d=128, x="bf16", causal=True, shape=3),
        # Images of several resolutions, text tokens with them, in one batch.
        dict(name="attention_packed 7 images", op="attention_packed", mode="self", b=7, low=300, high=4608,
             hq=24, hk=24, d=128, x="bf16", causal=False, shape=5),
        # The text encoder's head layout over short prompts.
        dict(name="attention_packed 96 short prompts", op="attention_packed", mode="self", b=96, low=1, high=509,
             hq=64, hk=64, d=64, x="f16", causal=False, shape=2),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear_s8", "qk_norm_rope", "attention_packed"])
    if op == "linear_s8":
        while True:
            m, n, k = _log(rng, 1, 4608), _log(rng, 256, 21504), _log(rng, 256, 15360)
            if rng.random() < 0.7:  # most layers are as wide as a multiple of 64; the rest is what it is
                n, k = (n + 63) // 64 * 64, (k + 63) // 64 * 64
            if m * n * k <= MOST_MACS:
                break
        x = rng.choice(["bf16", "bf16", "f16", "f32", "s8"])
        return dict(op=op, m=m, n=n, k=k, x=x, out=rng.choice(["bf16", "f32"] if x == "s8" else ["bf16", "f16"]),
                    act=rng.choice(["none", "gelu", "silu"]), bias=rng.random() < 0.7)
    if op == "qk_norm_rope":
        d, axes = rng.choice([(64, "64"), (64, "16,24,24"), (96, "32,64"), (128, "128"), (128, "16,56,56"),
                              (128, "32,48,48"), (128, "64"), (256, "256")])
        hk = rng.choice([1, 2, 4, 8, 12, 24])
        hq = hk * rng.choice([1, 2, 4]) if hk < 24 else 24
        t = _log(rng, 1, max(1, min(32768, MOST_VALUES // ((hq + hk) * d))))
        return dict(op=op, t=t, hq=hq, hk=hk, d=d, axes=axes, pairs=rng.choice(["neighbours", "halves"]),
                    x=rng.choice(["bf16", "f16", "f32"]), out=rng.choice(["bf16", "f16"]), norm=rng.random() < 0.8,
                    top=rng.choice([64, 8000]))
    mode = rng.choice(["cache", "self", "self"])
    d = rng.choice([64, 128, 128])
    hk = rng.choice([1, 2, 8, 12, 24])
    hq = hk * rng.choice([1, 2, 3, 4, 8]) if hk < 24 else 24
    while True:
        b = _log(rng, 1, 96)
        high = _log(rng, 16, 8192)
        case = dict(op=op, mode=mode, b=b, low=rng.choice([0, 1, (high + 2) // 3]), high=high, hq=hq, hk=hk, d=d,
                    x=rng.choice(["bf16", "bf16", "f16"]), causal=mode == "cache" or rng.random() < 0.5,
                    shape=rng.randrange(1000))
        ql, kl = _lengths(case)
        if hq * b * max(ql) * max(kl) <= MOST_SCORES and b * max(kl) * hk <= MOST_CACHE * 8 and sum(ql) and sum(kl):
            return case


def _lengths(case):
    """The sequences' query and key lengths: part of the case, the same for every seed.  The longest is always there."""
    rng = random.Random(case["shape"])
    low, high, b = case["low"], case["high"], case["b"]
    k = [min(high, _log(rng, max(1, low), high)) for _ in range(b)]
    k[rng.randrange(b)] = high
    if low == 0 and b > 1:
        k[rng.randrange(b)] = 0
    if case["mode"] == "cache":
        return [1] * b, k
    return list(k), k


# ---------------------------------------------------------------------------- inputs

def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + 17)
    s = {"case": case}
    if case["op"] == "linear_s8":
        m, n, k = case["m"], case["n"], case["k"]
        # Activations after a norm: unit scale, tokens of uneven size, a few channels far larger than the rest.
        x = _normal(g, m, k) * torch.exp(0.5 * _normal(g, m, 1))
        x[:, torch.randint(0, k, (max(1, k // 256),), generator=g, device=DEV)] *= 8.0
        pad = (k + 15) // 16 * 16  # 16-byte rows: 8-bit operands are laid out so when they are stored
        w = torch.zeros((n, pad), dtype=torch.int8, device=DEV)
        w[:, :k] = torch.clamp(torch.round(_normal(g, n, k, scale=127.0 / 4.0)), -127, 127).to(torch.int8)
        s["w"], s["w_scale"] = w[:, :k], 0.02 * 4.0 / 127.0 * torch.exp(0.1 * _normal(g, n))
        s["bias"] = _normal(g, n, scale=0.02) if case["bias"] else None
        if case["x"] == "s8":
            a = x.abs().amax(1, keepdim=True).clamp_min(1e-20)
            q = torch.zeros((m, pad), dtype=torch.int8, device=DEV)
            q[:, :k] = torch.round(x * (127.0 / a)).to(torch.int8)
            s["x"], s["x_scale"] = q[:, :k], (a / 127.0)[:, 0].contiguous()
        else:
            s["x"], s["x_scale"] = x.to(TYPES[case["x"]]), None
        return s
    if case["op"] == "qk_norm_rope":
        t, hq, hk, d = case["t"], case["hq"], case["hk"], case["d"]
        axes = [int(a) for a in case["axes"].split(",")]
        qkv = _normal(g, t, (hq + 2 * hk) * d).to(TYPES[case["x"]])  # [q | k | v] of each token, as the projection leaves it
        s["q"] = qkv[:, :hq * d].view(t, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
        s["axes"] = axes
        # Positions as the model has them: whole numbers, or halves of them where an image was resized.
        s["pos"] = torch.randint(0, 2 * case["top"], (t, len(axes)), generator=g, device=DEV).float() / 2
        s["qn"] = 1.0 + _normal(g, d, scale=0.1) if case["norm"] else None
        s["kn"] = 1.0 + _normal(g, d, scale=0.1) if case["norm"] else None
        return s
    ql, kl = _lengths(case)
    hq, hk, d, dt = case["hq"], case["hk"], case["d"], TYPES[case["x"]]
    tq, tk = sum(ql), sum(kl)
    if case["mode"] == "self":  # q, k and v are parts of one buffer
        qkv = _normal(g, tq, (hq + 2 * hk) * d).to(dt)
        s["q"] = qkv[:, :hq * d].view(tq, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hk) * d].view(tk, hk, d)
        s["v"] = qkv[:, (hq + hk) * d:].view(tk, hk, d)
    else:                       # caches of keys and of values
        s["q"] = _normal(g, tq, hq, d).to(dt)
        s["k"], s["v"] = _normal(g, tk, hk, d).to(dt), _normal(g, tk, hk, d).to(dt)
    # Normed heads meet in scores of a few units.
    s["q"].mul_(1.5)
    ends = lambda ls: torch.tensor([0] + [sum(ls[:i + 1]) for i in range(len(ls))], dtype=torch.int32, device=DEV)  # noqa: E731
    s["cu_q"], s["cu_k"] = ends(ql), ends(kl)
    s["max_q"], s["max_k"] = max(ql), max(kl)
    return s


# ---------------------------------------------------------------------------- one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    root = os.path.join(os.getcwd(), "chroma-radiance_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import b2g

    c = s["case"]
    if c["op"] == "linear_s8":
        return b2g.gemm_s8(s["x"], s["w"], s["w_scale"], s["bias"], out_dtype=TYPES[c["out"]], epilogue=c["act"],
                           x_scale=s["x_scale"])
    if c["op"] == "qk_norm_rope":
        return b2g.qk_norm_rope(s["q"], s["k"], s["pos"], s["axes"], q_norm=s["qn"], k_norm=s["kn"], eps=EPS,
                                interleaved=c["pairs"] == "neighbours", out_dtype=TYPES[c["out"]])
    return b2g.attention_packed(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=c["causal"])


def _run_plain(s):
    return {"linear_s8": _plain_linear, "qk_norm_rope": _plain_norm_rope,
            "attention_packed": _plain_attention}[s["case"]["op"]](s)


def _plain_linear(s):
    c, x = s["case"], s["x"].float()
    if s["x_scale"] is None:
        top = x.abs().amax(1, keepdim=True)
        some = top > 0
        x = torch.where(some, torch.round(x * 127.0 / torch.where(some, top, 1.0)), 0.0)
        scale = torch.where(some, top / 127.0, 1.0)
    else:
        scale = s["x_scale"][:, None]
    y = (x @ s["w"].float().t()) * scale * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    elif c["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    return y.to(TYPES[c["out"]])


def _plain_norm_rope(s):
    c = s["case"]
    turn = torch.cat([torch.arange(a // 2, device=DEV, dtype=torch.float32) * (-2.0 / a) for a in s["axes"]])
    which = torch.repeat_interleave(torch.arange(len(s["axes"]), device=DEV),
                                    torch.tensor([a // 2 for a in s["axes"]], device=DEV))
    angle = s["pos"][:, which] * torch.exp(turn * math.log(10000.0))
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    rot = 2 * cos.shape[-1]

    def one(x, w):
        x = x.float()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        if c["pairs"] == "neighbours":
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([y, x[..., rot:]], -1).to(TYPES[c["out"]])

    return one(s["q"], s["qn"]), one(s["k"], s["kn"])


def _plain_attention(s):
    c, cq, ck = s["case"], s["cu_q"].long(), s["cu_k"].long()
    hq, hk, d = c["hq"], c["hk"], c["d"]
    lq, lk = cq[1:] - cq[:-1], ck[1:] - ck[:-1]
    iq, ik = torch.arange(s["max_q"], device=DEV), torch.arange(s["max_k"], device=DEV)
    in_q, in_k = iq < lq[:, None], ik < lk[:, None]                       # [sequence, place]
    row_q = torch.where(in_q, cq[:-1, None] + iq, 0)
    row_k = torch.where(in_k, ck[:-1, None] + ik, 0)
    q = s["q"].float()[row_q].view(-1, s["max_q"], hk, hq // hk, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = (t.float()[row_k].transpose(1, 2) for t in (s["k"], s["v"]))   # [sequence, key head, place, d]
    score = (q @ k.transpose(2, 3)).mul_(d ** -0.5).view(-1, hk, hq // hk, s["max_q"], s["max_k"])
    sees = in_k[:, None, :].expand(-1, s["max_q"], -1)
    if c["causal"]:
        sees = sees & (ik <= (iq + (lk - lq)[:, None])[..., None])
    score = score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    y = (p.flatten(2, 3) @ v).view(*p.shape[:-1], d) / torch.where(total > 0, total, 1.0)
    y = y.permute(0, 3, 1, 2, 4).reshape(-1, s["max_q"], hq, d)[in_q]
    return y.to(TYPES[c["x"]])


# ---------------------------------------------------------------------------- work and definition

def work(case):
    if case["op"] == "linear_s8":
        m, n, k = case["m"], case["n"], case["k"]
        given = m * k * BYTES[case["x"]] + (4 * m if case["x"] == "s8" else 0)
        return {"bytes": given + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * BYTES[case["out"]],
                "flops": 2 * m * n * k}
    if case["op"] == "qk_norm_rope":
        values = case["t"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": values * (BYTES[case["x"]] + BYTES[case["out"]]) + 4 * case["t"] * len(case["axes"].split(",")),
                "flops": 8 * values}
    ql, kl = _lengths(case)
    seen = sum(sum(min(k, max(0, i + 1 + k - q)) for i in range(q)) if case["causal"] else q * k for q, k in zip(ql, kl))
    size = BYTES[case["x"]] * case["d"]
    return {"bytes": size * (2 * case["hq"] * sum(ql) + 2 * case["hk"] * sum(kl)), "flops": 4 * case["hq"] * case["d"] * seen}


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "linear_s8":
        if s["x_scale"] is not None:
            codes, unit = s["x"].to(f), s["x_scale"].to(f)
        else:
            x = s["x"].to(f)
            top = x.abs().max(dim=1).values
            unit = torch.where(top == 0, torch.ones_like(top), top / 127)
            codes = torch.round(torch.where(top[:, None] == 0, torch.zeros_like(x), x * 127 / top[:, None]))
        y = torch.mm(codes, s["w"].to(f).T) * unit.unsqueeze(1) * s["w_scale"].to(f).unsqueeze(0)
        if s["bias"] is not None:
            y += s["bias"].to(f)
        if case["act"] == "gelu":  # the tanh form as y times a logistic function
            y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        if case["act"] == "silu":
            y = y / (1 + torch.exp(-y))
        return y
    if case["op"] == "qk_norm_rope":
        def turned(x, w):
            x = x.to(f).clone()
            if w is not None:
                x *= (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).pow(-0.5)
                x *= w.to(f)
            rot, base = sum(s["axes"]), 0
            for axis, width in enumerate(s["axes"]):
                for j in range(width // 2):
                    pair = base + j
                    lo, hi = (2 * pair, 2 * pair + 1) if case["pairs"] == "neighbours" else (pair, pair + rot // 2)
                    z = torch.polar(torch.ones(x.shape[0], dtype=f, device=DEV),
                                    s["pos"][:, axis].to(f) * 10000.0 ** (-2 * j / width))
                    z = torch.complex(x[..., lo], x[..., hi]) * z[:, None]
                    x[..., lo], x[..., hi] = z.real, z.imag
                base += width // 2
            return x
        return turned(s["q"], s["qn"]), turned(s["k"], s["kn"])
    ql, kl = _lengths(case)
    if sum(a * b for a, b in zip(ql, kl)) * case["hq"] * case["d"] > 4e11:
        return None
    y = torch.zeros((sum(ql), case["hq"], case["d"]), dtype=f, device=DEV)
    group, q0, k0 = case["hq"] // case["hk"], 0, 0
    for nq, nk in zip(ql, kl):
        if nq and nk:
            for h in range(case["hk"]):
                k, v = s["k"][k0:k0 + nk, h].to(f), s["v"][k0:k0 + nk, h].to(f)
                q = s["q"][q0:q0 + nq, h * group:(h + 1) * group].to(f).transpose(0, 1)
                z = torch.matmul(q, k.T) / math.sqrt(case["d"])
                if case["causal"]:
                    hidden = torch.ones((nq, nk), dtype=torch.bool, device=DEV).triu(nk - nq + 1)
                    z[:, hidden] = -math.inf
                y[q0:q0 + nq, h * group:(h + 1) * group] = torch.matmul(torch.softmax(z, -1), v).nan_to_num(0.0).transpose(0, 1)
        q0, k0 = q0 + nq, k0 + nk
    return y
