"""Cases of the language-model row operators: block norms with their gate, residual scale and dropout
(forward and backward), dropout by itself, rotary positions and the rules applied to logits before a token
is chosen.  Where ``own`` is false, ``run`` computes them with elementary torch operations in 32 bits; where
it is true, through ``matrix_b200.lm``.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
M32 = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a decode step through the norms around a block: latency
        norm("norm decode", 1, 1, 4096, "bf16", gate="none", drop=0.0, save=False),
        # a training step's block: norms, a gate per channel, dropout in the residual branch
        norm("norm train", 4, 2048, 8192, "bf16", gate="channel", drop=0.1),
        # odd width and rows, float32, a gate of its own for every token
        norm("norm ragged f32", 1, 1111, 2001, "f32", gate="token", drop=0.0),
        # the backward pass of a training step
        norm("norm backward", 4, 2048, 4096, "bf16", gate="channel", drop=0.1, backward=True),
        # the backward pass with a gate per sequence (conditioned blocks), rows that do not divide evenly
        norm("norm backward ragged f16", 3, 1025, 1000, "f16", gate="sequence", drop=0.0, backward=True),
        # dropout of a block's hidden activations in training
        dict(name="dropout train", op="dropout", rows=16384, width=8192, type="bf16", drop=0.1),
        # odd sizes, float32
        dict(name="dropout ragged f32", op="dropout", rows=1001, width=4099, type="f32", drop=0.5),
        # a decode step of 64 sequences at positions far into a long context
        rotary("rotary decode", 64, 1, 32, 8, 128, 128, "bf16", positions=131072, scaled=True),
        # the gradient through the rotation of a training step's queries and keys
        rotary("rotary backward", 4, 4096, 32, 8, 128, 128, "bf16", positions=4096, interleaved=True, inverse=True),
        # a part of the head rotated, heads stored before tokens, odd length
        rotary("rotary partial f32", 2, 1023, 16, 16, 80, 32, "f32", positions=100000, heads_first=True),
        # one sequence's next token: every rule, a long history
        logits("logits one row", 1, 32768, "f32", history=1000, biases=64, mask=True),
        # a serving batch with a large vocabulary
        logits("logits batch", 256, 131072, "bf16", history=2048, biases=16, mask=True),
    ]


def norm(name, batch, length, width, type, gate, drop, save=True, backward=False, post=True, next=True, scale=1.0):
    c = dict(op="norm", batch=batch, length=length, width=width, type=type, gate=gate, drop=drop, save=save,
             backward=backward, post=post, next=next, scale=scale)
    return dict(c, name=name) if name else c


def rotary(name, batch, length, q_heads, k_heads, head, part, type, positions, interleaved=False, inverse=False,
           scaled=False, heads_first=False):
    c = dict(op="rotary", batch=batch, length=length, q_heads=q_heads, k_heads=k_heads, head=head, part=part,
             type=type, positions=positions, interleaved=interleaved, inverse=inverse, scaled=scaled,
             heads_first=heads_first)
    return dict(c, name=name) if name else c


def logits(name, rows, vocab, type, history, biases, mask):
    c = dict(op="logits", rows=rows, vocab=vocab, type=type, history=history, biases=biases, mask=mask)
    return dict(c, name=name) if name else c


def spread(rng, low, high):
    """A whole number of low..high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "backward", "backward", "dropout", "rotary", "rotary", "logits", "logits"])
    t = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind in ("norm", "backward"):
        width = spread(rng, 64, 16384)
        if rng.random() < 0.5:
            width = max(64, width // 64 * 64)
        most = (1 << (25 if kind == "norm" else 24)) // (2 if t == "f32" else 1) // width
        rows = spread(rng, 1, min(16384, most))
        batch = spread(rng, 1, min(16, rows))
        return norm("", batch, max(1, rows // batch), width, t, rng.choice(["none", "channel", "sequence", "token"]),
                    rng.choice([0.0, 0.1, 0.25]), backward=kind == "backward", post=rng.random() < 0.8,
                    next=rng.random() < 0.8, scale=rng.choice([1.0, 0.5]))
    if kind == "dropout":
        width = spread(rng, 1, 16384)
        rows = spread(rng, 1, min(65536, (1 << 25) // width))
        return dict(op="dropout", rows=rows, width=width, type=t, drop=rng.choice([0.05, 0.1, 0.5]))
    if kind == "rotary":
        head = rng.choice([64, 80, 96, 128, 192, 256])
        part = rng.choice([head, head // 2, 32])
        k_heads = rng.choice([1, 2, 4, 8])
        q_heads = k_heads * rng.choice([1, 2, 4, 7])
        length = 1 if rng.random() < 0.3 else spread(rng, 2, 8192)
        most = (1 << 25) // (length * (q_heads + k_heads) * head)
        return rotary("", spread(rng, 1, max(1, min(256 if length == 1 else 16, most))), length, q_heads, k_heads,
                      head, part, t, rng.choice([8192, 131072, 1000000]), rng.random() < 0.5, rng.random() < 0.5,
                      rng.random() < 0.5, rng.random() < 0.5)
    vocab = spread(rng, 1000, 262144)
    return logits("", spread(rng, 1, min(512, (1 << 24) // vocab)), vocab, t, spread(rng, 1, 4096), spread(rng, 1, 300),
                  rng.random() < 0.5)


# ------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]
    s = {"case": case, "seed": (seed * 0x9E3779B97F4A7C15) % (1 << 63), "offset": seed * 5 + (1 << 33)}

    def normal(*shape, mean=0.0, std=1.0, type=t):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(type)

    if case["op"] == "norm":
        b, n, d = case["batch"], case["length"], case["width"]
        s["branch"] = normal(b, n, d, std=0.5)
        s["residual"] = normal(b, n, d, std=2.0)  # forward: the stream before the block; backward: after it
        s["post_weight"] = normal(d, mean=1.0, std=0.1) if case["post"] else None
        s["next_weight"] = normal(d, mean=1.0, std=0.1) if case["next"] else None
        shape = {"none": None, "channel": (d,), "sequence": (b, 1, d), "token": (b, n, d)}[case["gate"]]
        s["gate"] = normal(*shape, mean=0.5, std=0.3) if shape else None
        if case["backward"]:
            s["d_residual"] = normal(b, n, d, std=0.1)
            s["d_normed"] = normal(b, n, d, std=0.1) if case["next"] else None
            for name, of in (("post", "branch"), ("next", "residual")):  # as the forward pass keeps them
                x = s[of].double()
                s[name + "_rstd"] = (x.square().mean(-1) + EPS).rsqrt().float().reshape(-1) if case[name] else None
    elif case["op"] == "dropout":
        s["x"] = normal(case["rows"], case["width"])
    elif case["op"] == "rotary":
        b, n, h = case["batch"], case["length"], case["head"]
        for name, heads in (("q", case["q_heads"]), ("k", case["k_heads"])):
            s[name] = normal(b, heads, n, h).transpose(1, 2) if case["heads_first"] else normal(b, n, heads, h)
        first = torch.randint(0, max(1, case["positions"] - n), (b, 1), generator=g, device="cuda")
        s["positions"] = (first + torch.arange(n, device="cuda")).to(torch.int32)
        # the angular frequencies, laid out once by a user's program; "scaled" interpolates the slow ones
        # (fewer than 1 turn over the first 4096 positions by 32, those of 32 turns or more not at all)
        r = case["part"]
        theta = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
        s["scale"] = 1.0
        if case["scaled"]:
            keep = ((4096 * theta / (2 * math.pi) - 1) / 31).clamp(0, 1)
            theta = theta * keep + theta / 32 * (1 - keep)
            s["scale"] = 0.1 * math.log(32) + 1
        s["theta"] = theta.cuda()
    else:
        n, v, length, k = case["rows"], case["vocab"], case["history"], case["biases"]
        s["logits"] = normal(n, v, std=3.0)

        def some(*shape):  # tokens: a few common ones, many rare ones
            return (torch.rand(*shape, generator=g, device="cuda").pow(3) * v).to(torch.int32).clamp_(max=v - 1)

        def upto(m):
            return torch.randint(0, m + 1, (n,), generator=g, device="cuda", dtype=torch.int32)

        s["tokens"] = some(n, length)
        s["lengths"] = torch.maximum(upto(length), torch.tensor(length // 2, device="cuda", dtype=torch.int32))
        s["prompt_lengths"] = torch.minimum(upto(length // 2), s["lengths"])
        s["repetition"] = torch.rand(n, generator=g, device="cuda") + 1.0
        s["frequency"] = torch.rand(n, generator=g, device="cuda")
        s["presence"] = torch.rand(n, generator=g, device="cuda")
        s["bias_tokens"] = some(n, k)
        s["bias_values"] = torch.randn(n, k, generator=g, device="cuda") * 4
        s["mask"] = None
        if case["mask"]:
            s["mask"] = torch.randint(-(1 << 31), 1 << 31, (n, (v + 31) // 32), generator=g, device="cuda").to(torch.int32)
            if n > 3:
                s["mask"][n // 2] = 0  # a grammar that has ended: no token is allowed
    return s


# ------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------
_lm = None


def lm():
    global _lm
    if _lm is None:
        from matrix_b200 import backend, lm as module

        backend.init(torch.cuda.current_device())
        _lm = module
    return _lm


def run(s):
    c = s["case"]
    if own:
        return run_own(s, c)
    if c["op"] == "norm":
        return plain_norm_backward(s, c) if c["backward"] else plain_norm(s, c)
    return {"dropout": plain_dropout, "rotary": plain_rotary, "logits": plain_logits}[c["op"]](s, c)


def run_own(s, c):
    if c["op"] == "norm":
        how = dict(post_weight=s["post_weight"], gate=s["gate"], next_weight=s["next_weight"],
                   residual_scale=c["scale"], branch_scale=0.5, dropout=c["drop"], seed=s["seed"], offset=s["offset"])
        if c["backward"]:
            g = lm().block_norm_backward(s["d_residual"], s["d_normed"], s["residual"], s["branch"],
                                         post_rstd=s["post_rstd"], next_rstd=s["next_rstd"], **how)
            return {"residual": g.residual, "branch": g.branch, "post_weight": g.post_weight, "gate": g.gate,
                    "next_weight": g.next_weight}
        o = lm().block_norm(s["residual"], s["branch"], eps=EPS, save_rstd=c["save"], **how)
        return {"residual": o.residual, "normed": o.normed, "post_rstd": o.post_rstd, "next_rstd": o.next_rstd}
    if c["op"] == "dropout":
        return lm().dropout(s["x"], c["drop"], s["seed"], s["offset"])
    if c["op"] == "rotary":
        return lm().rotary(s["q"], s["k"], s["positions"], s["theta"], scale=s["scale"],
                           interleaved=c["interleaved"], inverse=c["inverse"])
    return lm().logits_rules(s["logits"], tokens=s["tokens"], lengths=s["lengths"], prompt_lengths=s["prompt_lengths"],
                             repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                             bias_tokens=s["bias_tokens"], bias_values=s["bias_values"], mask=s["mask"])


def plain_philox(seed, offset, rows, width):
    """The 16-bit lanes of Philox4x32-10 for [rows, width]: counter (column / 8, row, offset), eight lanes each."""
    blocks = (width + 7) // 8
    c0 = torch.arange(blocks, device="cuda").expand(rows, blocks)
    c1 = torch.arange(rows, device="cuda")[:, None].expand(rows, blocks)
    c2 = torch.full_like(c0, offset & M32)
    c3 = torch.full_like(c0, offset >> 32)
    k0, k1 = seed & M32, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & M32) ^ c1 ^ k0, p1 & M32, ((p0 >> 32) & M32) ^ c3 ^ k1, p0 & M32
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    lanes = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], -1)
    return lanes.reshape(rows, blocks * 8)[:, :width]


def plain_keep(p, seed, offset, rows, width):
    """What a kept element is multiplied by, and 0 where it is dropped."""
    kept = round((1 - p) * 65536)
    return (plain_philox(seed, offset, rows, width) < kept).float() * (65536 / kept)


def plain_dropout(s, c):
    return (s["x"].float() * plain_keep(c["drop"], s["seed"], s["offset"], c["rows"], c["width"])).to(s["x"].dtype)


def plain_norm(s, c):
    x, b = s["residual"].float(), s["branch"].float()
    post_rstd = next_rstd = normed = None
    if c["post"]:
        post_rstd = (b.square().mean(-1, keepdim=True) + EPS).rsqrt()
        b = b * post_rstd * s["post_weight"].float()
    if c["drop"]:
        b = b * plain_keep(c["drop"], s["seed"], s["offset"], c["batch"] * c["length"], c["width"]).view(b.shape)
    if s["gate"] is not None:
        b = b * s["gate"].float()
    h = c["scale"] * x + 0.5 * b
    if c["next"]:
        next_rstd = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
        normed = (h * next_rstd * s["next_weight"].float()).to(s["residual"].dtype)
    return {"residual": h.to(s["residual"].dtype), "normed": normed,
            "post_rstd": post_rstd.reshape(-1) if c["post"] and c["save"] else None,
            "next_rstd": next_rstd.reshape(-1) if c["next"] and c["save"] else None}


def plain_norm_backward(s, c):
    h, b, dh = s["residual"].float(), s["branch"].float(), s["d_residual"].float()
    d_post = d_next = d_gate = None
    if c["next"]:
        r = s["next_rstd"].view(c["batch"], c["length"], 1)
        da = s["d_normed"].float()
        p = da * s["next_weight"].float()
        d_next = (da * h * r).sum((0, 1))
        dh = dh + r * p - h * r.pow(3) * (p * h).mean(-1, keepdim=True)
    q = 0.5 * dh
    if c["drop"]:
        q = q * plain_keep(c["drop"], s["seed"], s["offset"], c["batch"] * c["length"], c["width"]).view(q.shape)
    unit = b
    if c["post"]:
        r = s["post_rstd"].view(c["batch"], c["length"], 1)
        unit = b * r
    if s["gate"] is not None:
        dg = q * unit
        if c["post"]:
            dg = dg * s["post_weight"].float()
        d_gate = {"channel": lambda: dg.sum((0, 1)), "sequence": lambda: dg.sum(1, keepdim=True),
                  "token": lambda: dg}[c["gate"]]().to(s["gate"].dtype)
        q = q * s["gate"].float()
    if c["post"]:
        d_post = (q * unit).sum((0, 1))
        q = q * s["post_weight"].float()
        q = r * q - unit * r * (q * unit).mean(-1, keepdim=True)
    t = s["residual"].dtype
    return {"residual": (c["scale"] * dh).to(t), "branch": q.to(t), "post_weight": d_post, "gate": d_gate,
            "next_weight": d_next}


def plain_rotary(s, c):
    # the angle in 64 bits: in 32 its error at the positions of a long context is larger than the results'
    angle = s["positions"].double()[..., None] * s["theta"]
    cos, sin = (f(angle).float()[:, :, None] * s["scale"] for f in (torch.cos, torch.sin))
    if c["inverse"]:
        sin = -sin
    return [plain_rotate(s["q"], cos, sin, c), plain_rotate(s["k"], cos, sin, c)]


def plain_rotate(x, cos, sin, c):
    r = c["part"]
    y = x[..., :r].float()
    if c["interleaved"]:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = y[..., : r // 2], y[..., r // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y.to(x.dtype), x[..., r:]], -1)


def plain_logits(s, c):
    n, v = c["rows"], c["vocab"]
    x = s["logits"].float()
    at = torch.arange(c["history"], device="cuda")[None]
    told = at < s["lengths"][:, None]
    made = told & (at >= s["prompt_lengths"][:, None])
    tokens = s["tokens"].long()
    seen = torch.zeros(n, v, device="cuda").scatter_add_(1, tokens, told.float())
    count = torch.zeros(n, v, device="cuda").scatter_add_(1, tokens, made.float())
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    # of several biases for a token the last one of the list counts
    entry = torch.arange(1, c["biases"] + 1, device="cuda").expand(n, -1)
    last = torch.zeros(n, v, dtype=torch.long, device="cuda").scatter_reduce_(1, s["bias_tokens"].long(), entry, "amax")
    x = x + torch.where(last > 0, s["bias_values"].gather(1, (last - 1).clamp(min=0)), 0.0)
    if s["mask"] is not None:
        ids = torch.arange(v, device="cuda")
        x = torch.where((s["mask"][:, ids // 32] >> (ids % 32)) & 1 > 0, x, -math.inf)
    return x.to(s["logits"].dtype)


# ------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    c, e = case, SIZE[case["type"]]
    if c["op"] == "norm":
        rows, d = c["batch"] * c["length"], c["width"]
        gate = {"none": 0, "channel": d, "sequence": c["batch"] * d, "token": rows * d}[c["gate"]]
        n = rows * d
        rstd = 4 * rows * (c["post"] + c["next"])
        if c["backward"]:  # reads d_residual, d_normed, residual, branch; writes two gradients, the gate's, the weights'
            used = 2 + c["next"] + (c["post"] or gate > 0)
            return {"bytes": e * ((used + 2) * n + 2 * gate) + (e + 4) * d * (c["post"] + c["next"]) + rstd,
                    "flops": 24 * n}
        return {"bytes": e * ((3 + c["next"]) * n + gate + d * (c["post"] + c["next"])) + rstd * c["save"],
                "flops": 12 * n}
    if c["op"] == "dropout":
        return {"bytes": 2 * e * c["rows"] * c["width"], "flops": c["rows"] * c["width"]}
    if c["op"] == "rotary":
        n = c["batch"] * c["length"] * (c["q_heads"] + c["k_heads"])
        return {"bytes": 2 * e * n * c["head"] + 4 * c["batch"] * c["length"] + 4 * c["part"], "flops": 3 * n * c["part"]}
    n = c["rows"] * c["vocab"]
    # half the history at least is filled; lists of biases and lengths; one bit a token where there is a mask
    lists = c["rows"] * (3 * c["history"] + 8 * c["biases"] + 20)
    return {"bytes": 2 * e * n + lists + (c["rows"] * ((c["vocab"] + 31) // 32) * 4 if c["mask"] else 0), "flops": 6 * n}


# ------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": exact_norm, "dropout": exact_dropout, "rotary": exact_rotary, "logits": exact_logits}[case["op"]](s, case)


def exact_mulhi(a, m):
    """The upper and lower 32 bits of a * m, through products of 16 bits."""
    a0, a1, m0, m1 = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
    mid = a1 * m0 + ((a0 * m0) >> 16)
    mid2 = a0 * m1 + (mid & 0xFFFF)
    return a1 * m1 + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | ((a0 * m0) & 0xFFFF)


def exact_mask(p, seed, offset, rows, width):
    """keep / keep probability in 64 bits, in slabs of rows."""
    kept = round((1 - p) * 65536)
    out = torch.empty(rows, width, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 22) // width)
    block = torch.arange((width + 7) // 8, device="cuda")
    for r in range(0, rows, step):
        row = torch.arange(r, min(rows, r + step), device="cuda")
        word = [block[None] + 0 * row[:, None], row[:, None] + 0 * block[None],
                torch.full((len(row), len(block)), offset % (1 << 32), device="cuda"),
                torch.full((len(row), len(block)), offset >> 32, device="cuda")]
        for i in range(10):
            k0, k1 = (seed + i * 0x9E3779B9) & M32, ((seed >> 32) + i * 0xBB67AE85) & M32
            (h0, l0), (h1, l1) = exact_mulhi(word[0], 0xD2511F53), exact_mulhi(word[2], 0xCD9E8D57)
            word = [h1 ^ word[1] ^ k0, l1, h0 ^ word[3] ^ k1, l0]
        lane = torch.empty(len(row), len(block), 8, dtype=torch.long, device="cuda")
        for i in range(4):
            lane[:, :, 2 * i], lane[:, :, 2 * i + 1] = word[i] % 65536, word[i] // 65536
        out[r:r + len(row)] = torch.where(lane.view(len(row), -1)[:, :width] < kept, 65536 / kept, 0.0)
    return out


def exact_dropout(s, c):
    return s["x"].double() * exact_mask(c["drop"], s["seed"], s["offset"], c["rows"], c["width"])


def exact_norm(s, c):
    def double(v):
        return None if v is None else v.double().requires_grad_(c["backward"])

    def unit(v):
        return v * (v.square().mean(-1, keepdim=True) + EPS).rsqrt()

    with torch.set_grad_enabled(c["backward"]):
        x, b, g, wp, wn = (double(s[k]) for k in ("residual", "branch", "gate", "post_weight", "next_weight"))
        n = b if wp is None else unit(b) * wp
        if c["drop"]:
            n = n * exact_mask(c["drop"], s["seed"], s["offset"], c["batch"] * c["length"], c["width"]).view(n.shape)
        if g is not None:
            n = n * g
        if not c["backward"]:
            h = c["scale"] * x + 0.5 * n
            rstd = [(v.square().mean(-1) + EPS).rsqrt().reshape(-1) if has and c["save"] else None
                    for v, has in ((b, c["post"]), (h, c["next"]))]
            return {"residual": h, "normed": None if wn is None else unit(h) * wn, "post_rstd": rstd[0],
                    "next_rstd": rstd[1]}
        # the gradient at the stream after the block, then through the branch
        total = s["d_residual"].double()
        dn = None
        if wn is not None:
            dx, dn = torch.autograd.grad(unit(x) * wn, [x, wn], s["d_normed"].double())
            total = total + dx
        wanted = [v for v in (b, wp, g) if v is not None]
        got = iter(torch.autograd.grad(0.5 * n, wanted, total))
        db, dp, dg = (next(got) if v is not None else None for v in (b, wp, g))
        return {"residual": c["scale"] * total, "branch": db, "post_weight": dp, "gate": dg, "next_weight": dn}


def exact_rotary(s, c):
    angle = s["positions"].double()[:, :, None] * s["theta"]
    turn = torch.polar(torch.full_like(angle, s["scale"]), -angle if c["inverse"] else angle)[:, :, None]
    out = []
    for x in (s["q"], s["k"]):
        y, r = x.double().clone(), c["part"]
        even = slice(0, r, 2) if c["interleaved"] else slice(0, r // 2)
        odd = slice(1, r, 2) if c["interleaved"] else slice(r // 2, r)
        z = torch.complex(y[..., even].contiguous(), y[..., odd].contiguous()) * turn
        y[..., even], y[..., odd] = z.real, z.imag
        out.append(y)
    return out


def exact_logits(s, c):
    x = s["logits"].double()
    v = c["vocab"]
    for i, (n, p) in enumerate(zip(s["lengths"].tolist(), s["prompt_lengths"].tolist())):
        t = s["tokens"][i, :n].long()
        seen = torch.bincount(t, minlength=v) > 0
        count = torch.bincount(t[p:], minlength=v).double()
        r = s["repetition"][i].double()
        row = x[i]
        row = torch.where(seen, torch.where(row > 0, row / r, row * r), row)
        row = row - s["frequency"][i].double() * count - s["presence"][i].double() * (count > 0)
        bias = dict(zip(s["bias_tokens"][i].tolist(), s["bias_values"][i].tolist()))
        row[list(bias)] += torch.tensor(list(bias.values()), dtype=torch.float64, device="cuda")
        if s["mask"] is not None:
            bits = (s["mask"][i][:, None] >> torch.arange(32, device="cuda", dtype=torch.int32)[None]) & 1
            row[bits.reshape(-1)[:v] == 0] = -math.inf
        x[i] = row
    return x
