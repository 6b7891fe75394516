"""Measured cases of the packed batch's further operators: each request's own low-rank adapter beside a shared
projection, and attention over key blocks that a cheap score selects.

A case is one pass through one operator.  `run` computes it either in plain form (elementary torch
operations in 32 bits, rounded once at the end) or, with `own` set, through the engine's entry points
in chroma-radiance_b200/b2g.py.  `exact` states each operator's definition in 64 bits.

    lora              out = act(y + s_r (x A_r^T) B_r^T) for the rows of request r, s_r, A_r, B_r its adapter's scale and
                      matrices; gated_residual: y + gate * (..); a request without an adapter keeps act(y)
    block_means       the mean of each block of 128 keys of a sequence (the last one may be shorter), per key head; with
                      `since`, of those blocks alone that hold a key from there on
    select_blocks     per tile of 128 queries of a sequence and key head, one bit per key block: the first and the last few
                      blocks in sight, those that some query of the tile sees in part, and the `top` best others by
                      (sum of the tile's queries, all heads of the group) . (mean of the block)
    attention_blocks  softmax(q k^T scale) v within each sequence over the keys of the chosen blocks
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
BLOCK = 128  # keys of a block, queries of a tile
#: what one pass may cost at most: the largest listed case of each operator
MOST_LORA = 13938 * (3072 + 2 * 9216)  # values read and written
MOST_LORA_MACS = 13938 * 16 * (3072 + 9216)
MOST_KEYS = 16384 * 24 * 128           # values of k
MOST_SCORES = 128 * 128 * 24 * 28 * 128  # query heads x queries x chosen keys, whole blocks


# ---------------------------------------------------------------------------- cases

def listed():
    return [
        # One token of each of 48 requests, 48 adapters: latency, the adapters are all there is to read.
        dict(name="lora 48 single tokens 4096 to 4096", op="lora", b=48, low=1, high=1, shape=1, k=4096, n=4096, r=16,
             adapters=64, x="bf16", y="bf16", act="none"),
        # Five images of different sizes with their prompts, an adapter each, beside the block's q, k and v.
        dict(name="lora 5 requests 3072 to 9216", op="lora", b=5, low=700, high=4608, shape=11, k=3072, n=9216, r=16,
             adapters=5, x="bf16", y="bf16", act="none"),
        # A text encoder's feed-forward over a few prompts (odd row counts, fp16, GELU), adapters of rank 64.
        dict(name="lora 9 prompts 4096 to 10240 gelu", op="lora", b=9, low=3, high=253, shape=4, k=4096, n=10240, r=64,
             adapters=4, x="f16", y="f16", act="gelu"),
        # The block's second layer at 512^2 into the F32 residual stream, two requests.
        dict(name="lora 2 requests 15360 to 3072 gated residual", op="lora", b=2, low=1300, high=1536, shape=6, k=15360,
             n=3072, r=32, adapters=3, x="bf16", y="f32", act="gated_residual"),
        # The newest key of 48 caches: the block it belongs to.
        dict(name="block_means newest key of 48 caches", op="block_means", mode="cache", b=48, low=1, high=16383, queries=1,
             hk=8, d=128, x="bf16", shape=7, since=True),
        # All keys of a 2048^2 image, 24 heads, k read from the fused projection.
        dict(name="block_means 16384 tokens", op="block_means", mode="self", b=1, low=16384, high=16384, hq=24, hk=24,
             d=128, x="bf16", shape=0, since=False),
        # One query for each of 48 caches of uneven fill, grouped heads.
        dict(name="select_blocks 48 single queries", op="select_blocks", mode="cache", b=48, low=1, high=16383, queries=1,
             hq=32, hk=8, d=128, x="bf16", causal=True, top=16, first=1, last=1, shape=7),
        # A 2048^2 image: its prompt's blocks (the first four) always, 24 of the others.
        dict(name="select_blocks 16384 tokens", op="select_blocks", mode="self", b=1, low=16384, high=16384, hq=24, hk=24,
             d=128, x="bf16", causal=False, top=24, first=4, last=0, shape=0),
        # The same caches: 18 blocks of up to 128.
        dict(name="attention_blocks 48 single queries", op="attention_blocks", mode="cache", b=48, low=1, high=16383,
             queries=1, hq=32, hk=8, d=128, x="bf16", causal=True, top=16, first=1, last=1, shape=7),
        # Causal prompts from a word to some pages, grouped heads of 64 values, fp16.
        dict(name="attention_blocks 12 causal prompts", op="attention_blocks", mode="self", b=12, low=1, high=4095, hq=32,
             hk=8, d=64, x="f16", causal=True, top=6, first=1, last=2, shape=3),
        # Three 1024^2 images, 13 of 36 blocks.
        dict(name="attention_blocks 3 images of 4608", op="attention_blocks", mode="self", b=3, low=4608, high=4608, hq=24,
             hk=24, d=128, x="bf16", causal=False, top=9, first=4, last=0, shape=0),
        # A 2048^2 image, 28 of 128 blocks.
        dict(name="attention_blocks 16384 tokens", op="attention_blocks", mode="self", b=1, low=16384, high=16384, hq=24,
             hk=24, d=128, x="bf16", causal=False, top=24, first=4, last=0, shape=0),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["lora", "lora", "block_means", "select_blocks", "attention_blocks", "attention_blocks"])
    if op == "lora":
        while True:
            high = _log(rng, 1, 4608)
            case = dict(op=op, b=_log(rng, 1, 64), low=rng.choice([0, 1, high]), high=high, shape=rng.randrange(1000),
                        k=8 * _log(rng, 32, 1920), n=_log(rng, 64, 21504), r=rng.choice([8, 16, 16, 32, 64, 128]),
                        adapters=_log(rng, 1, 64), x=rng.choice(["bf16", "bf16", "f16"]))
            case["act"] = rng.choice(["none", "none", "gelu", "silu", "gated_residual"])
            case["y"] = "f32" if case["act"] == "gated_residual" else rng.choice([case["x"], case["x"], "f32"])
            if rng.random() < 0.7:  # most layers are as wide as a multiple of 64; the rest is what it is
                case["k"], case["n"] = (case["k"] + 63) // 64 * 64, (case["n"] + 63) // 64 * 64
            rows = sum(_lengths(case)[0])
            if 0 < rows and rows * (case["k"] + 2 * case["n"]) <= MOST_LORA and \
                    rows * case["r"] * (case["k"] + case["n"]) <= MOST_LORA_MACS:
                return case
    mode = rng.choice(["cache", "self", "self"])
    d = rng.choice([64, 128, 128])
    hk = rng.choice([1, 2, 8, 12, 24])
    hq = hk * rng.choice([1, 2, 3, 4, 8]) if hk < 24 else 24
    while True:
        high = _log(rng, 16, 16384)
        case = dict(op=op, mode=mode, b=_log(rng, 1, 96), low=rng.choice([0, 1, (high + 2) // 3]), high=high, hq=hq, hk=hk,
                    d=d, x=rng.choice(["bf16", "bf16", "f16"]), shape=rng.randrange(1000))
        if mode == "cache":
            case["queries"] = rng.choice([1, 1, 1, 2, 5])
        if op == "block_means":
            case["since"] = mode == "cache" and rng.random() < 0.5
        else:
            case.update(causal=mode == "cache" or rng.random() < 0.5, top=_log(rng, 1, 32), first=rng.choice([0, 1, 4]),
                        last=rng.choice([0, 1, 2]))
        ql, kl, room = _lengths(case)
        if not sum(kl) or sum(room) * hk * d > MOST_KEYS:
            continue
        if op == "attention_blocks" and sum(-(-q // BLOCK) for q in ql) * BLOCK * hq * _most_chosen(case) * BLOCK > MOST_SCORES:
            continue
        if op == "select_blocks" and sum(-(-q // BLOCK) for q in ql) * hk * -(-max(room) // BLOCK) * d > 128 * 24 * 128 * 128:
            continue
        if mode == "self" and sum(ql) * hq * d > 2 * MOST_KEYS:
            continue
        return case


def _lengths(case):
    """The sequences' query and key lengths and the rows that their keys have room for: part of the case, the same for
    every seed.  The longest is always there.  For lora the first is the requests' rows."""
    rng = random.Random(case["shape"])
    low, high, b = case["low"], case["high"], case["b"]
    k = [min(high, _log(rng, max(1, low), high)) for _ in range(b)]
    k[rng.randrange(b)] = high
    if low == 0 and b > 1:
        k[rng.randrange(b)] = 0
    if case.get("mode") == "cache":
        return [case["queries"]] * b, k, [-(-n // 256) * 256 for n in k]
    return list(k), k, list(k)


def _sight(case, q, k, tile):
    """The keys that a tile's first and last query see."""
    last = min(q, (tile + 1) * BLOCK) - 1
    if not case["causal"]:
        return k, k
    return tuple(max(0, min(k, i + 1 + k - q)) for i in (tile * BLOCK, last))


def _count(case, q, k, tile):
    """How many blocks a tile takes: part of the case."""
    first, last = _sight(case, q, k, tile)
    nb = -(-last // BLOCK)
    sure = sum(j < case["first"] or j >= nb - case["last"] or min((j + 1) * BLOCK, last) > first for j in range(nb))
    return min(nb, sure + case["top"])


def _most_chosen(case):
    ql, kl, _ = _lengths(case)
    return max([1] + [_count(case, q, k, t) for q, k in set(zip(ql, kl)) for t in range(-(-q // BLOCK))])


# ---------------------------------------------------------------------------- inputs

def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _ends(ls):
    at = [0]
    for n in ls:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + 29)
    s = {"case": case}
    dt = TYPES[case["x"]]
    if case["op"] == "lora":
        rows, _, _ = _lengths(case)
        m, k, n, r, many = sum(rows), case["k"], case["n"], case["r"], case["adapters"]
        s["x"] = _normal(g, m, k, dtype=dt)
        s["a"] = _normal(g, many, r, k, scale=k ** -0.5, dtype=dt)
        s["b"] = _normal(g, many, n, r, scale=0.25 * r ** -0.5, dtype=dt)
        s["scale"] = torch.exp(0.5 * _normal(g, many))
        # Every request asks for some adapter; one in ten has none (never all of them).
        ids = torch.randint(0, many, (case["b"],), generator=g, device=DEV)
        none = torch.rand(case["b"], generator=g, device=DEV) < 0.1
        none[0] = False
        s["ids"] = torch.where(none, -1, ids).int()
        s["cu"], s["most"], s["rows"] = _ends(rows), max(rows), m
        s["y"] = _normal(g, m, n, dtype=TYPES[case["y"]])
        s["gate"] = _normal(g, n, scale=0.5) if case["act"] == "gated_residual" else None
        return s
    ql, kl, room = _lengths(case)
    hk, d, tq, tk = case["hk"], case["d"], sum(ql), sum(room)
    hq = case.get("hq", hk)
    s["cu_q"], s["cu_k"] = _ends(ql), _ends(room)
    s["lens"] = torch.tensor(kl, dtype=torch.int32, device=DEV) if case["mode"] == "cache" else None
    s["max_q"], s["max_k"] = max(ql), max(room)
    s["blocks"], s["tiles"] = sum(-(-n // BLOCK) for n in room), sum(-(-n // BLOCK) for n in ql)
    # Neighbouring keys are alike: a part that a run of 64 shares.
    near = lambda t, h: _normal(g, -(-t // 64) or 1, h, d, scale=0.5).repeat_interleave(64, 0)[:t]  # noqa: E731
    if case["op"] == "select_blocks":
        s["q"] = (_normal(g, tq, hq, d) + near(tq, hq)).to(dt)
        # The keys' means as block_means leaves them, blocks without a key zero.
        means = _normal(g, tk // BLOCK + case["b"], hk, d, scale=0.5)
        used = torch.zeros(tk // BLOCK + case["b"], dtype=torch.bool, device=DEV)
        at = 0
        for n, have in zip(room, kl):
            used[at:at + -(-have // BLOCK)] = True
            at += -(-n // BLOCK)
        s["means"] = means * used[:, None, None]
        return s
    if case["mode"] == "self":  # q, k and v are parts of one buffer
        qkv = _normal(g, tq, (hq + 2 * hk) * d)
        qkv[:, :(hq + hk) * d] += near(tq, hq + hk).flatten(1)
        qkv = qkv.to(dt)
        s["q"] = qkv[:, :hq * d].view(tq, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hk) * d].view(tk, hk, d)
        s["v"] = qkv[:, (hq + hk) * d:].view(tk, hk, d)
    else:                       # caches of keys and of values
        s["k"] = (_normal(g, tk, hk, d) + near(tk, hk)).to(dt)
        if case["op"] == "attention_blocks":
            s["q"], s["v"] = _normal(g, tq, hq, d, dtype=dt), _normal(g, tk, hk, d, dtype=dt)
    if case["op"] == "block_means":
        # The means of earlier steps; this step has written the last `queries` keys.
        s["means"] = _normal(g, tk // BLOCK + case["b"], hk, d, scale=0.5)
        s["since"] = (s["lens"] - case["queries"]).clamp_min(0).int() if case["since"] else None
        return s
    # Blocks as a selection leaves them, from random scores.
    words = -(-(-(-s["max_k"] // BLOCK)) // 32)
    s["most"] = _most_chosen(case)
    rule = _tiles(s)
    score = torch.rand((s["tiles"], hk, 32 * words), generator=g, device=DEV, dtype=torch.float64)
    s["chosen"] = _pack(_taken(case, rule, score))
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
    if c["op"] == "lora":
        return b2g.lora(s["x"], s["a"], s["b"], s["y"], s["cu"], ids=s["ids"], scale=s["scale"], epilogue=c["act"],
                        gate=s["gate"])
    if c["op"] == "block_means":
        return b2g.block_means(s["k"], s["cu_k"], k_lens=s["lens"], since=s["since"],
                               out=s["means"] if c["since"] else None)
    if c["op"] == "select_blocks":
        return b2g.select_blocks(s["q"], s["means"], s["cu_q"], c["top"], cu_k=s["cu_k"], k_lens=s["lens"], first=c["first"],
                                 last=c["last"], causal=c["causal"], max_k=s["max_k"])
    return b2g.attention_blocks(s["q"], s["k"], s["v"], s["chosen"], s["cu_q"], cu_k=s["cu_k"], k_lens=s["lens"],
                                causal=c["causal"])


def _run_plain(s):
    return {"lora": _plain_lora, "block_means": _plain_means, "select_blocks": _plain_select,
            "attention_blocks": _plain_attention}[s["case"]["op"]](s)


def _plain_lora(s):
    c, cu = s["case"], s["cu"].long()
    place = torch.arange(s["most"], device=DEV)
    live = place < (cu[1:] - cu[:-1])[:, None]
    row = torch.where(live, cu[:-1, None] + place, 0)
    has = s["ids"] >= 0
    which = torch.where(has, s["ids"], 0).long()
    t = torch.matmul(s["x"].float()[row], s["a"].float()[which].transpose(1, 2))
    delta = torch.matmul(t, s["b"].float()[which].transpose(1, 2)) * (s["scale"][which] * has)[:, None, None]
    delta = delta[live]
    y = s["y"].float()
    if c["act"] == "gated_residual":
        return (y + s["gate"] * delta).to(s["y"].dtype)
    y = y + delta
    if c["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    elif c["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    return y.to(s["y"].dtype)


def _plain_means(s):
    c, cu = s["case"], s["cu_k"].long()
    room = cu[1:] - cu[:-1]
    lens = room if s["lens"] is None else s["lens"].long()
    many = (room + BLOCK - 1) // BLOCK
    base = torch.cumsum(many, 0) - many
    if s["since"] is None:
        seq = torch.repeat_interleave(torch.arange(c["b"], device=DEV), many, output_size=s["blocks"])
        j = torch.arange(s["blocks"], device=DEV) - base[seq]
    else:  # the blocks that a sequence's last keys touch
        touched = 1 + (c["queries"] + BLOCK - 2) // BLOCK
        seq = torch.arange(c["b"], device=DEV).repeat_interleave(touched)
        j = (s["since"].long()[:, None] // BLOCK + torch.arange(touched, device=DEV)).flatten()
    live = j[:, None] * BLOCK + torch.arange(BLOCK, device=DEV) < lens[seq][:, None]
    row = torch.where(live, (cu[:-1][seq] + j * BLOCK)[:, None] + torch.arange(BLOCK, device=DEV), 0)
    mean = (s["k"][row].float() * live[..., None, None]).sum(1) / live.sum(1).clamp_min(1)[:, None, None]
    if s["since"] is None:
        return torch.cat([mean, mean.new_zeros((s["means"].shape[0] - s["blocks"], *mean.shape[1:]))])
    # (blocks without a key go to a row past the end)
    out = torch.cat([s["means"], s["means"][:1]])
    out[torch.where(live.any(1), base[seq] + j, s["means"].shape[0])] = mean
    return s["means"].copy_(out[:-1])


def _tiles(s):
    """Per tile: its sequence, its first row, the sequence's lengths, the keys that its first and last query see."""
    c, cq, ck = s["case"], s["cu_q"].long(), s["cu_k"].long()
    lq = cq[1:] - cq[:-1]
    lk = ck[1:] - ck[:-1] if s["lens"] is None else s["lens"].long()
    many = (lq + BLOCK - 1) // BLOCK
    seq = torch.repeat_interleave(torch.arange(len(lq), device=DEV), many, output_size=s["tiles"])
    row = (torch.arange(s["tiles"], device=DEV) - (torch.cumsum(many, 0) - many)[seq]) * BLOCK
    q, k = lq[seq], lk[seq]
    if c["causal"]:
        first = (row + 1 + k - q).clamp_min(0).minimum(k)
        last = (torch.minimum(row + BLOCK, q) + k - q).clamp_min(0).minimum(k)
    else:
        first = last = k
    return {"seq": seq, "row": row, "q": q, "k": k, "first": first, "last": last}


def _taken(c, t, score):
    """The rule of select_blocks on scores [tile, key head, block]."""
    j = torch.arange(score.shape[-1], device=DEV)
    nb = ((t["last"] + BLOCK - 1) // BLOCK)[:, None]
    inside = j < nb
    part = torch.minimum((j + 1) * BLOCK, t["last"][:, None]) > t["first"][:, None]
    sure = inside & ((j < c["first"]) | (j >= nb - c["last"]) | part)
    free = inside & ~sure
    order = score.masked_fill(~free[:, None], -math.inf).sort(dim=-1, descending=True, stable=True).indices
    best = torch.zeros(score.shape, dtype=torch.bool, device=DEV)
    best.scatter_(-1, order[..., :c["top"]], True)
    return sure[:, None] | (best & free[:, None])


def _pack(bits):
    """[.., 32 words] truth values -> [.., words] int32, block j being bit j % 32 of word j / 32."""
    w = (bits.unflatten(-1, (-1, 32)).long() << torch.arange(32, device=DEV)).sum(-1)
    return (w - ((w >> 31) << 32)).int()


def _plain_select(s):
    c, t = s["case"], _tiles(s)
    hk, d, nb = c["hk"], c["d"], -(-s["max_k"] // BLOCK)
    words = (nb + 31) // 32
    place = torch.arange(min(BLOCK, s["max_q"]), device=DEV)
    live = t["row"][:, None] + place < t["q"][:, None]
    row = torch.where(live, (s["cu_q"].long()[:-1][t["seq"]] + t["row"])[:, None] + place, 0)
    heads = s["q"].double().unflatten(1, (hk, c["hq"] // hk)).sum(2)
    pooled = (heads[row] * live[..., None, None]).sum(1)                      # [tile, key head, d]
    room = s["cu_k"].long()[1:] - s["cu_k"].long()[:-1]
    many = (room + BLOCK - 1) // BLOCK
    base = torch.cumsum(many, 0) - many
    at = torch.minimum(base[t["seq"]][:, None] + torch.arange(nb, device=DEV), torch.tensor(s["means"].shape[0] - 1, device=DEV))
    score = torch.matmul(s["means"].double()[at].transpose(1, 2), pooled[..., None])[..., 0]  # [tile, key head, block]
    score = torch.nn.functional.pad(score, (0, 32 * words - nb))
    chosen = _pack(_taken(c, t, score))
    out = chosen.new_zeros((s["q"].shape[0] // BLOCK + c["b"], hk, words))  # (as many tiles as there can be)
    out[:s["tiles"]] = chosen
    return out


def _plain_attention(s):
    c, t = s["case"], _tiles(s)
    hq, hk, d, n = c["hq"], c["hk"], c["d"], s["most"]
    bits = (s["chosen"][..., None] >> torch.arange(32, device=DEV)).bitwise_and(1).flatten(-2) > 0
    block = bits.int().sort(dim=-1, descending=True, stable=True).indices[..., :n]            # [tile, key head, n]
    taken = torch.arange(n, device=DEV) < bits.sum(-1, keepdim=True)
    key = (block[..., None] * BLOCK + torch.arange(BLOCK, device=DEV)).flatten(2)         # [tile, key head, n 128]
    live_k = taken.repeat_interleave(BLOCK, -1) & (key < t["k"][:, None, None])
    row_k = torch.where(live_k, s["cu_k"].long()[:-1][t["seq"]][:, None, None] + key, 0)
    high = min(BLOCK, s["max_q"])
    index = t["row"][:, None] + torch.arange(high, device=DEV)
    live_q = index < t["q"][:, None]
    row_q = torch.where(live_q, s["cu_q"].long()[:-1][t["seq"]][:, None] + index, 0)
    q = s["q"][row_q].float().unflatten(2, (hk, hq // hk)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    head = torch.arange(hk, device=DEV)[None, :, None]
    score = torch.matmul(q, s["k"][row_k, head].float().transpose(2, 3)).mul_(d ** -0.5).unflatten(2, (hq // hk, high))
    sees = live_k[:, :, None]
    if c["causal"]:
        sees = sees & (key[:, :, None] <= (index + (t["k"] - t["q"])[:, None])[:, None, :, None])
    score = score.masked_fill_(~sees[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.flatten(2, 3), s["v"][row_k, head].float()).unflatten(2, (hq // hk, high))
    y = y / torch.where(total > 0, total, 1.0)
    return y.permute(0, 3, 1, 2, 4).reshape(-1, high, hq, d)[live_q].to(TYPES[c["x"]])


# ---------------------------------------------------------------------------- work and definition

def work(case):
    if case["op"] == "lora":
        rows, _, _ = _lengths(case)
        m, k, n, r, some = sum(rows), case["k"], case["n"], case["r"], min(case["b"], case["adapters"])
        return {"bytes": BYTES[case["x"]] * (m * k + some * r * (k + n)) + 2 * BYTES[case["y"]] * m * n,
                "flops": 2 * m * r * (k + n)}
    ql, kl, room = _lengths(case)
    hk, d, size = case["hk"], case["d"], BYTES[case["x"]]
    if case["op"] == "block_means":
        keys, blocks = sum(kl), sum(-(-n // BLOCK) for n in room)
        if case["since"]:  # of each cache the blocks that hold its last keys
            firsts = [max(0, k - case["queries"]) // BLOCK for k in kl]
            keys, blocks = sum(k - f * BLOCK for k, f in zip(kl, firsts)), sum(-(-k // BLOCK) - f for k, f in zip(kl, firsts))
        return {"bytes": keys * hk * d * size + 4 * blocks * hk * d, "flops": keys * hk * d}
    tiles = [(q, k, t) for q, k in zip(ql, kl) for t in range(-(-q // BLOCK))]
    if case["op"] == "select_blocks":
        pairs = sum(-(-_sight(case, *x)[1] // BLOCK) for x in tiles)
        blocks = sum(-(-k // BLOCK) for k in kl)
        return {"bytes": sum(ql) * case["hq"] * d * size + 4 * blocks * hk * d + len(tiles) * hk * (max(room) // 1024 + 1) * 4,
                "flops": 2 * pairs * hk * d + sum(ql) * case["hq"] * d}
    chosen = [min(_count(case, *x) * BLOCK, _sight(case, *x)[1]) for x in tiles]
    seen = sum(n * min(BLOCK, q - t * BLOCK) for n, (q, _, t) in zip(chosen, tiles))
    # Keys: of a sequence at most all of them, at most what its tiles choose.
    keys = sum(min(k, sum(n for n, x in zip(chosen, tiles) if x[:2] == (q, k)) // max(1, list(zip(ql, kl)).count((q, k))))
               for q, k in zip(ql, kl))
    return {"bytes": size * d * (2 * case["hq"] * sum(ql) + 2 * hk * keys) + 4 * len(tiles) * hk * (max(room) // 4096 + 1),
            "flops": 4 * case["hq"] * d * seen}


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "lora":
        y = s["y"].to(f)
        delta, at = torch.zeros_like(y), 0
        for n, i in zip(_lengths(case)[0], s["ids"].tolist()):
            if i >= 0:
                low = torch.mm(s["x"][at:at + n].to(f), s["a"][i].to(f).T)
                delta[at:at + n] = torch.mm(low, s["b"][i].to(f).T) * float(s["scale"][i])
            at += n
        if case["act"] == "gated_residual":
            return y + s["gate"].to(f) * delta
        y += delta
        if case["act"] == "gelu":  # the tanh form as y times a logistic function
            y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        if case["act"] == "silu":
            y = y / (1 + torch.exp(-y))
        return y
    ql, kl, room = _lengths(case)
    hk, d, group = case["hk"], case["d"], case.get("hq", case["hk"]) // case["hk"]
    if case["op"] == "block_means":
        out, at, k0 = s["means"].to(f) if case["since"] else torch.zeros_like(s["means"], dtype=f), 0, 0
        for n, have in zip(room, kl):
            since = max(0, have - case["queries"]) if case["since"] else 0
            for j in range(since // BLOCK, -(-have // BLOCK)):
                out[at + j] = s["k"][k0 + j * BLOCK:k0 + min(have, (j + 1) * BLOCK)].to(f).mean(0)
            at += -(-n // BLOCK)
            k0 += n
        return out
    if case["op"] == "select_blocks":
        words = -(-(-(-max(room) // BLOCK)) // 32)
        out = torch.zeros((sum(ql) // BLOCK + case["b"], hk, words), dtype=torch.int64)
        tile, q0, at = 0, 0, 0
        for q, k, n in zip(ql, kl, room):
            for t in range(-(-q // BLOCK)):
                first, last = _sight(case, q, k, t)
                nb = -(-last // BLOCK)
                sure = [j < case["first"] or j >= nb - case["last"] or min((j + 1) * BLOCK, last) > first for j in range(nb)]
                tile_q = s["q"][q0 + t * BLOCK:q0 + min(q, (t + 1) * BLOCK)].to(f)
                for h, score in enumerate(torch.einsum("rhgd,bhd->hb", tile_q.view(-1, hk, group, d), s["means"][at:at + nb].to(f)).tolist()):
                    free = sorted((j for j in range(nb) if not sure[j]), key=lambda j: (-score[j], j))[:case["top"]]  # noqa: B023
                    for j in free + [j for j in range(nb) if sure[j]]:
                        out[tile, h, j // 32] |= 1 << j % 32
                tile += 1
            q0 += q
            at += -(-n // BLOCK)
        return torch.where(out >= 1 << 31, out - (1 << 32), out).int().to(DEV)
    y = torch.zeros((sum(ql), hk * group, d), dtype=f, device=DEV)
    bits, tile, q0, k0 = s["chosen"].cpu(), 0, 0, 0
    for q, k, n in zip(ql, kl, room):
        tiles = -(-q // BLOCK)
        if q and k:
            mine = ((bits[tile:tile + tiles, :, :, None] >> torch.arange(32)) & 1).flatten(2).bool()  # [tile, head, block]
            for h in range(hk):
                hidden = ~mine[:, h].to(DEV).repeat_interleave(BLOCK, 0)[:q].repeat_interleave(BLOCK, 1)[:, :k]
                if case["causal"]:
                    hidden = hidden | torch.ones((q, k), dtype=torch.bool, device=DEV).triu(k - q + 1)
                keys, values = s["k"][k0:k0 + k, h].to(f), s["v"][k0:k0 + k, h].to(f)
                for i in range(h * group, (h + 1) * group):
                    z = torch.matmul(s["q"][q0:q0 + q, i].to(f), keys.T) / math.sqrt(d)
                    y[q0:q0 + q, i] = torch.matmul(torch.softmax(z.masked_fill_(hidden, -math.inf), -1), values).nan_to_num(0.0)
        tile += tiles
        q0 += q
        k0 += n
    return y
