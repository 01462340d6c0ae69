"""Cases of the attention operators of a language model: the norms of queries and keys for each head with their
rotation (forward and backward), a paged cache of keys and values written and read back (quantised or not), the
attention of one new token over it, and the attention of whole prompts.  Where ``own`` is false, ``run`` computes them
with elementary torch operations in 32 bits; where it is true, through ``matrix_b200.lm``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
LARGEST = 448.0  # of e4m3


# ------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------
def listed():
    return [
        # a decode step of 64 sequences far into a long context: latency
        heads("heads decode", 64, 1, 32, 8, 128, 128, "bf16", positions=131072, scaled=True, save=False),
        # the queries and keys of a training step
        heads("heads train", 4, 4096, 32, 8, 128, 128, "bf16", positions=4096),
        # their gradients, with those of the two weights
        heads("heads backward", 4, 4096, 32, 8, 128, 128, "bf16", positions=4096, backward=True),
        # a part of the head rotated, interleaved pairs, odd length, float32
        heads("heads backward ragged f32", 2, 1023, 16, 16, 80, 32, "f32", positions=100000, interleaved=True, backward=True),
        # the keys and values of a decode step of 64 sequences, quantised
        cache("cache decode", 64, 8, 128, "bf16", page=16, small=True),
        # those of a long prompt, quantised as they are written, and a prefix as long read back
        cache("cache prompt", 16384, 8, 128, "bf16", page=64, small=True),
        # one sequence's next token: latency
        decode("decode one", 1, 1500, 32, 8, 128, "bf16", page=16),
        # a serving batch of sequences of different lengths
        decode("decode batch", 64, 8192, 32, 8, 128, "bf16", page=64),
        # few sequences with a long context, the cache in 8 bits, an odd group of heads
        decode("decode long e4m3", 4, 131072, 56, 8, 128, "f16", page=16, small=True),
        # two long prompts
        prompt("prompt long", 2, 8192, 32, 8, 128, "bf16"),
        # many short prompts of odd lengths behind a cached prefix
        prompt("prompt ragged f16", 24, 777, 16, 4, 64, "f16", prefix=300),
        # float32, a head that is no power of two
        prompt("prompt f32", 3, 500, 8, 2, 80, "f32"),
    ]


def heads(name, batch, length, q_heads, k_heads, head, part, type, positions, interleaved=False, scaled=False,
          backward=False, save=True):
    c = dict(op="heads", batch=batch, length=length, q_heads=q_heads, k_heads=k_heads, head=head, part=part, type=type,
             positions=positions, interleaved=interleaved, scaled=scaled, backward=backward, save=save)
    return dict(c, name=name) if name else c


def cache(name, tokens, heads, head, type, page, small):
    c = dict(op="cache", tokens=tokens, heads=heads, head=head, type=type, page=page, small=small)
    return dict(c, name=name) if name else c


def decode(name, batch, length, q_heads, k_heads, head, type, page, small=False):
    c = dict(op="decode", batch=batch, length=length, q_heads=q_heads, k_heads=k_heads, head=head, type=type, page=page,
             small=small)
    return dict(c, name=name) if name else c


def prompt(name, sequences, length, q_heads, k_heads, head, type, prefix=0):
    c = dict(op="prompt", sequences=sequences, length=length, q_heads=q_heads, k_heads=k_heads, head=head, type=type,
             prefix=prefix)
    return dict(c, name=name) if name else c


def spread(rng, low, high):
    """A whole number of low..high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["heads", "heads", "cache", "decode", "decode", "prompt", "prompt"])
    t = rng.choice(["f32", "f16", "bf16", "bf16"])
    head = rng.choice([64, 80, 96, 128, 128, 192, 256])
    k_heads = rng.choice([1, 2, 4, 8])
    q_heads = k_heads * rng.choice([1, 2, 4, 7, 8])
    if kind == "heads":
        length = 1 if rng.random() < 0.3 else spread(rng, 2, 8192)
        most = (1 << 25) // (length * (q_heads + k_heads) * head)
        return heads("", spread(rng, 1, max(1, min(256 if length == 1 else 16, most))), length, q_heads, k_heads, head,
                     rng.choice([head, head // 2, 32]), t, rng.choice([8192, 131072, 1000000]), rng.random() < 0.5,
                     rng.random() < 0.5, rng.random() < 0.5)
    if kind == "cache":
        return cache("", spread(rng, 1, (1 << 24) // (k_heads * head)), k_heads, head, t, rng.choice([1, 16, 24, 64, 128]),
                     rng.random() < 0.7)
    if kind == "decode":
        small = rng.random() < 0.4
        length = spread(rng, 1, 131072)
        most = (1 << 29) // (length * k_heads * head * (1 if small else SIZE[t]))
        return decode("", spread(rng, 1, max(1, min(256, most))), length, q_heads, k_heads, head, t,
                      rng.choice([16, 24, 64, 128]), small)
    limit = (1 << (38 if t != "f32" else 33)) // (q_heads * head)
    length = spread(rng, 1, min(8192, math.isqrt(limit)))
    prefix = rng.choice([0, 0, spread(rng, 1, 2048)])
    prefix = min(prefix, (limit // length - length) // 2)
    return prompt("", spread(rng, 1, max(1, min(64, limit // (length * (length + 2 * prefix))))), length, q_heads, k_heads,
                  head, t, prefix)


# ------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------
def lengths_of(case):
    """The lengths of a case's sequences: the longest first, the others between an eighth of it and it."""
    n = case["batch"] if case["op"] == "decode" else case["sequences"]
    rng = random.Random(case["length"] * 1009 + n)
    return [case["length"]] + [rng.randint(max(1, case["length"] // 8), case["length"]) for _ in range(n - 1)]


def prefixes_of(case):
    rng = random.Random(case["prefix"] * 31 + case["sequences"])
    return [rng.randint(0, case["prefix"]) for _ in range(case["sequences"])]


def starts_of(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def pages_like(pages, page, heads, head, type):
    """Keys or values of a cache: [pages, slots, heads, head], the slots of a head next to each other in memory."""
    return torch.empty(pages, heads, page, head, device="cuda", dtype=type).transpose(1, 2)


def new_cache(pages, page, heads, head, t, small):
    """Keys, values and, of a cache in 8 bits, the exponents of their scales."""
    kinds = [torch.float8_e4m3fn if small else t] * 2
    out = [pages_like(pages, page, heads, head, kind) for kind in kinds]
    if small:
        out += [torch.zeros(pages, heads, page, device="cuda", dtype=torch.int8).transpose(1, 2) for _ in kinds]
    else:
        out += [None, None]
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]
    s = {"case": case}

    def normal(*shape, mean=0.0, std=1.0, type=t):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(type)

    def some_heads(*shape, std=1.0):
        """Heads whose channels differ in size, as projections give them."""
        size = 0.5 + 1.5 * torch.rand(*shape[-2:], generator=g, device="cuda")
        x = torch.randn(*shape, generator=g, device="cuda")
        return x.mul_(size * std).to(t)

    if case["op"] == "heads":
        b, n, h = case["batch"], case["length"], case["head"]
        for name, count in (("q", case["q_heads"]), ("k", case["k_heads"])):
            s[name] = some_heads(b, n, count, h)
            s[name + "_weight"] = normal(h, mean=1.0, std=0.1)
            if case["backward"]:
                s["d_" + name] = normal(b, n, count, h, std=0.1)
                s[name + "_rstd"] = (s[name].double().square().mean(-1) + EPS).rsqrt().float()
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
    elif case["op"] == "cache":
        n, h, d, page = case["tokens"], case["heads"], case["head"], case["page"]
        pages = (n + page - 1) // page + 8
        s["cache"] = new_cache(pages, page, h, d, t, case["small"])
        s["k"], s["v"] = some_heads(n, h, d), some_heads(n, h, d, std=0.5)
        # pages in an order of their own, full ones first: a token's slot
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(n, device="cuda")
        s["slots"] = (order[at // page] * page + at % page).to(torch.int32)
    elif case["op"] == "decode":
        b, h, d, page = case["batch"], case["k_heads"], case["head"], case["page"]
        lengths = lengths_of(case)
        used = [(n + page - 1) // page for n in lengths]
        pages = sum(used) + 8
        s["q"] = some_heads(b, case["q_heads"], d)
        s["cache"] = new_cache(pages, page, h, d, t, case["small"])
        for x, std, e in ((s["cache"][0], 1.0, s["cache"][2]), (s["cache"][1], 0.5, s["cache"][3])):
            if e is None:
                # in pieces: a large cache in 32 bits would need twice its memory again
                for i in range(0, pages, 1024):
                    x[i:i + 1024] = torch.randn(x[i:i + 1024].shape, generator=g, device="cuda").mul_(std).to(t)
            else:
                for i in range(0, pages, 1024):
                    y = torch.randn(x[i:i + 1024].shape, generator=g, device="cuda").mul_(100.0).clamp_(-LARGEST, LARGEST)
                    x[i:i + 1024].view(torch.int8).copy_(y.to(torch.float8_e4m3fn).view(torch.int8))
                e.copy_(torch.randint(-8, -5, e.shape, generator=g, device="cuda").to(torch.int8))
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.zeros(b, max(used), dtype=torch.int32, device="cuda")
        first = 0
        for i, n in enumerate(used):
            table[i, :n] = order[first:first + n]
            first += n
        s["table"] = table
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    else:
        lengths = lengths_of(case)
        starts = starts_of(lengths)
        k_starts = starts_of([n + p for n, p in zip(lengths, prefixes_of(case))])
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["k_starts"] = torch.tensor(k_starts, dtype=torch.int32, device="cuda") if case["prefix"] else None
        s["q"] = some_heads(starts[-1], case["q_heads"], case["head"])
        s["k"] = some_heads(k_starts[-1], case["k_heads"], case["head"])
        s["v"] = some_heads(k_starts[-1], case["k_heads"], case["head"], std=0.5)
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
    if c["op"] == "heads":
        return plain_heads_backward(s, c) if c["backward"] else plain_heads(s, c)
    return {"cache": plain_cache, "decode": plain_decode, "prompt": plain_prompt}[c["op"]](s, c)


def run_own(s, c):
    if c["op"] == "heads":
        how = dict(q_weight=s["q_weight"], k_weight=s["k_weight"], scale=s["scale"], interleaved=c["interleaved"])
        if c["backward"]:
            g = lm().head_norm_rotary_backward(s["d_q"], s["d_k"], s["q"], s["k"], s["positions"], s["theta"],
                                               q_rstd=s["q_rstd"], k_rstd=s["k_rstd"], **how)
            return {"q": g.q, "k": g.k, "q_weight": g.q_weight, "k_weight": g.k_weight}
        o = lm().head_norm_rotary(s["q"], s["k"], s["positions"], s["theta"], eps=EPS, save_rstd=c["save"], **how)
        return {"q": o.q, "k": o.k, "q_rstd": o.q_rstd, "k_rstd": o.k_rstd}
    if c["op"] == "cache":
        pages = lm().KVCache(*s["cache"])
        lm().cache_write(pages, s["k"], s["v"], s["slots"])
        k, v = lm().cache_read(pages, s["slots"], dtype=s["k"].dtype)
        return {"k": k, "v": v}
    if c["op"] == "decode":
        return lm().decode_attention(s["q"], lm().KVCache(*s["cache"]), s["table"], s["lengths"])
    return lm().prompt_attention(s["q"], s["k"], s["v"], s["starts"], k_starts=s["k_starts"])


def plain_turn(x, s, c, sign):
    """The first `part` elements of the heads turned by their positions (sign -1: back)."""
    # the angle in 64 bits: in 32 its error at the positions of a long context is larger than the results'
    angle = s["positions"].double()[..., None] * s["theta"]
    cos, sin = (f(angle).float()[:, :, None] * s["scale"] for f in (torch.cos, torch.sin))
    r, sin = c["part"], sin * sign
    y = x[..., :r]
    if c["interleaved"]:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = y[..., : r // 2], y[..., r // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., r:]], -1)


def plain_heads(s, c):
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        out[name] = plain_turn(x * r * s[name + "_weight"].float(), s, c, 1.0).to(s[name].dtype)
        out[name + "_rstd"] = r[..., 0] if c["save"] else None
    return out


def plain_heads_backward(s, c):
    out = {}
    for name in ("q", "k"):
        x, r, w = s[name].float(), s[name + "_rstd"][..., None], s[name + "_weight"].float()
        g = plain_turn(s["d_" + name].float(), s, c, -1.0)
        out[name + "_weight"] = (g * x * r).sum((0, 1, 2))
        u = g * w
        out[name] = (r * u - x * r.pow(3) * (u * x).mean(-1, keepdim=True)).to(s[name].dtype)
    return out


def power_of_two(e):
    """2^e as floats, for whole e of -126 .. 127: by its bits, since a power function may round."""
    return ((e.int() + 127) << 23).view(torch.float32)


def plain_quantise(x):
    """Bytes of e4m3 and the exponent of the scale for each head: the least power of two that keeps the largest
    element within 448, so that neither the division nor the product that reads it back rounds."""
    top, exponent = torch.frexp(x.abs().amax(-1))  # top of 0.5 .. 1; 448 is 0.875 * 2^9
    e = torch.where(top > 0, exponent - 9 + (top > 0.875), 0).clamp(-96, 96)
    return (x * power_of_two(-e[..., None])).to(torch.float8_e4m3fn), e.to(torch.int8)


def plain_cache(s, c):
    out = {}
    page, slots = c["page"], s["slots"].long()
    where = (slots // page, slots % page)
    for name, to, exponents in (("k", s["cache"][0], s["cache"][2]), ("v", s["cache"][1], s["cache"][3])):
        if c["small"]:
            q, e = plain_quantise(s[name].float())
            to.view(torch.int8)[where] = q.view(torch.int8)
            exponents[where] = e
            back = to.view(torch.int8)[where].view(torch.float8_e4m3fn).float()
            out[name] = (back * power_of_two(exponents[where][..., None])).to(s[name].dtype)
        else:
            to[where] = s[name]
            out[name] = to[where].clone()
    return out


def plain_read(x, exponents, pages):
    """Keys or values of the pages [n] as floats [tokens, heads, head]."""
    if exponents is None:
        return x[pages].flatten(0, 1).float()
    y = x.view(torch.int8)[pages].view(torch.float8_e4m3fn).float()
    return (y * power_of_two(exponents[pages][..., None])).flatten(0, 1)


def plain_decode(s, c):
    keys, values, ke, ve = s["cache"]
    group, d = c["q_heads"] // c["k_heads"], c["head"]
    out = torch.empty_like(s["q"])
    for i in range(c["batch"]):
        k, v = plain_read(keys, ke, s["table"][i].long()), plain_read(values, ve, s["table"][i].long())
        q = s["q"][i].float().view(c["k_heads"], group, d)
        scores = q @ k.permute(1, 2, 0) / math.sqrt(d)
        told = torch.arange(len(k), device="cuda") < s["lengths"][i]
        scores = torch.where(told, scores, -math.inf)
        p = (scores - scores.amax(-1, keepdim=True)).exp()
        v = torch.where(told[:, None, None], v, 0.0)
        o = p @ v.transpose(0, 1) / p.sum(-1, keepdim=True)
        out[i] = o.reshape(c["q_heads"], d).to(out.dtype)
    return out


def plain_prompt(s, c):
    group, d = c["q_heads"] // c["k_heads"], c["head"]
    out = torch.empty_like(s["q"])
    lengths = lengths_of(c)
    starts = starts_of(lengths)
    k_starts = starts_of([n + p for n, p in zip(lengths, prefixes_of(c))])
    for i, n in enumerate(lengths):
        m = k_starts[i + 1] - k_starts[i]
        seen = torch.arange(m, device="cuda") <= torch.arange(n, device="cuda")[:, None] + (m - n)
        for h in range(c["k_heads"]):
            q = s["q"][starts[i]:starts[i + 1], h * group:(h + 1) * group].float().transpose(0, 1)
            k = s["k"][k_starts[i]:k_starts[i + 1], h].float()
            v = s["v"][k_starts[i]:k_starts[i + 1], h].float()
            scores = torch.where(seen, q @ k.T / math.sqrt(d), -math.inf)
            p = (scores - scores.amax(-1, keepdim=True)).exp()
            o = p @ v / p.sum(-1, keepdim=True)
            out[starts[i]:starts[i + 1], h * group:(h + 1) * group] = o.transpose(0, 1).to(out.dtype)
    return out


# ------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    c, e = case, SIZE[case["type"]]
    if c["op"] == "heads":
        tokens = c["batch"] * c["length"]
        n = tokens * (c["q_heads"] + c["k_heads"])
        small = 4 * tokens + 4 * c["part"] + 2 * e * c["head"] + 4 * n * (c["save"] or c["backward"])
        if c["backward"]:  # reads the gradients and the heads, writes their gradients and the weights'
            return {"bytes": 3 * e * n * c["head"] + small + 8 * c["head"], "flops": 16 * n * c["head"]}
        return {"bytes": 2 * e * n * c["head"] + small, "flops": 8 * n * c["head"]}
    if c["op"] == "cache":  # keys and values read and stored, and read back
        n = 2 * c["tokens"] * c["heads"]
        held = n * (c["head"] + 1) if c["small"] else n * c["head"] * e
        return {"bytes": 2 * (n * c["head"] * e + held) + 8 * c["tokens"], "flops": 4 * n * c["head"]}
    if c["op"] == "decode":
        tokens = sum(lengths_of(c))
        held = c["head"] + 1 if c["small"] else c["head"] * e
        ends = 2 * e * c["batch"] * c["q_heads"] * c["head"]
        return {"bytes": 2 * tokens * c["k_heads"] * held + ends + 4 * tokens // c["page"],
                "flops": 4 * tokens * c["q_heads"] * c["head"]}
    lengths, prefixes = lengths_of(c), prefixes_of(c)
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(lengths, prefixes))
    rows = 2 * sum(lengths) * c["q_heads"] + 2 * (sum(lengths) + sum(prefixes)) * c["k_heads"]
    return {"bytes": e * rows * c["head"], "flops": 4 * pairs * c["q_heads"] * c["head"]}


# ------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"heads": exact_heads, "cache": exact_cache, "decode": exact_decode, "prompt": exact_prompt}[case["op"]](s, case)


def exact_heads(s, c):
    turn = torch.polar(torch.tensor(s["scale"], dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, :, None] * s["theta"])[:, :, None]
    out, r = {}, c["part"]
    even = slice(0, r, 2) if c["interleaved"] else slice(0, r // 2)
    odd = slice(1, r, 2) if c["interleaved"] else slice(r // 2, r)
    for name in ("q", "k"):
        with torch.set_grad_enabled(c["backward"]):
            x = s[name].double().requires_grad_(c["backward"])
            w = s[name + "_weight"].double().requires_grad_(c["backward"])
            rstd = (x * x).mean(-1).add(EPS).pow(-0.5)
            n = x * rstd[..., None] * w
            z = torch.complex(n[..., even], n[..., odd]) * turn
            y = n.clone()
            y[..., even], y[..., odd] = z.real, z.imag
            if c["backward"]:
                out[name], out[name + "_weight"] = torch.autograd.grad(y, [x, w], s["d_" + name].double())
            else:
                out[name], out[name + "_rstd"] = y, rstd if c["save"] else None
    order = ("q", "k", "q_weight", "k_weight") if c["backward"] else ("q", "k", "q_rstd", "k_rstd")
    return {name: out[name] for name in order}


def exact_cache(s, c):
    out = {}
    for name in ("k", "v"):
        x = s[name].double()
        if c["small"]:
            e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / LARGEST)).clamp(-96, 96)
            y = x * torch.exp2(-e)
            # to 4 significant bits, or to multiples of 2^-9 below 2^-6
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            x = torch.round(y / step) * step * torch.exp2(e)
        out[name] = x
    return out


def exact_decode(s, c):
    group, page = c["q_heads"] // c["k_heads"], c["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lengths_of(c)):
        at = torch.arange(n, device="cuda")
        where = (s["table"][i].long()[at // page], at % page)
        kv = []
        for x, e in zip(s["cache"][:2], s["cache"][2:]):
            if e is None:
                kv.append(x[where].double())
            else:
                kv.append(x.view(torch.int8)[where].view(torch.float8_e4m3fn).double() * torch.exp2(e[where].double())[..., None])
        for h in range(c["k_heads"]):
            p = torch.softmax(s["q"][i, h * group:(h + 1) * group].double() @ kv[0][:, h].T * c["head"] ** -0.5, -1)
            out[i, h * group:(h + 1) * group] = p @ kv[1][:, h]
    return out


def exact_prompt(s, c):
    group = c["q_heads"] // c["k_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    first = k_first = 0
    for n, prefix in zip(lengths_of(c), prefixes_of(c)):
        hidden = torch.ones(n, n + prefix, dtype=torch.bool, device="cuda").triu(prefix + 1)
        for h in range(c["q_heads"]):
            k, v = (s[x][k_first:k_first + n + prefix, h // group].double() for x in "kv")
            scores = (s["q"][first:first + n, h].double() @ k.T * c["head"] ** -0.5).masked_fill_(hidden, -math.inf)
            out[first:first + n, h] = torch.softmax(scores, -1) @ v
        first, k_first = first + n, k_first + n + prefix
    return out
