"""Plain implementations of the language-model row operators in 64 bits, on the CPU, and the bounds that the
kernels' results are held to.

Bounds.  A result stored in a type of p significand bits is rounded once, by at most 2^-p of itself (float32
2^-24, float16 2^-11, bfloat16 2^-8; float16 below its normal range by at most 2^-25).  Before that the
arithmetic is in 32 bits, u = 2^-24: a sum of at most a few ten thousand terms, of which a thread adds a few
dozen one after another and a tree of depth 10 the rest, is off by less than 48 u of the sum of magnitudes, a
square root halves that, and about ten products and additions follow.  So every result is held to
    |got - exact| <= 2^-p |exact| + 2^-18 * magnitude                                    (2^-18 = 64 u)
where `magnitude` is the same formula with every term's absolute value.  A value whose rounding passes the
type's largest is stored as an infinity.
"""
from __future__ import annotations

import math

import numpy as np
import torch

ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-42, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38}
WORK = 2.0 ** -18
M32 = 0xFFFFFFFF


def assert_within(got: torch.Tensor, exact: torch.Tensor, magnitude: torch.Tensor, what: str, work: float = WORK) -> None:
    assert got.shape == exact.shape, f"{what}: shape {tuple(got.shape)} != {tuple(exact.shape)}"
    g = got.detach().cpu().double()
    tol = ROUND[got.dtype] * exact.abs() + work * magnitude + TINY[got.dtype]
    bad = ~((g - exact).abs() <= tol)
    bad &= ~((g == exact) | (torch.isnan(g) & torch.isnan(exact)))
    bad &= ~(torch.isinf(g) & (g.sign() == exact.sign()) & (exact.abs() + tol >= torch.finfo(got.dtype).max))
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {g.numel()} outside the bound; first {i}: got {g[i].item()!r}, "
                             f"exact {exact[i].item()!r}, bound {tol[i].item()!r}")


def philox(counter, key):
    """Philox4x32-10 of uint64 arrays holding 32-bit words."""
    c, k = [np.asarray(x, dtype=np.uint64) for x in counter], list(key)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        s, m = np.uint64(32), np.uint64(M32)
        c = [(p1 >> s) ^ c[1] ^ np.uint64(k[0]), p1 & m, (p0 >> s) ^ c[3] ^ np.uint64(k[1]), p0 & m]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return c


def lanes(seed: int, offset: int, rows: int, width: int) -> np.ndarray:
    blocks = (width + 7) // 8
    block, row = np.meshgrid(np.arange(blocks, dtype=np.uint64), np.arange(rows, dtype=np.uint64))
    one = np.ones_like(block)
    seed, offset = seed % (1 << 64), offset % (1 << 64)
    words = philox([block, row, one * np.uint64(offset & M32), one * np.uint64(offset >> 32)], [seed & M32, seed >> 32])
    out = np.empty((rows, blocks, 8), dtype=np.int64)
    for i, w in enumerate(words):
        out[:, :, 2 * i], out[:, :, 2 * i + 1] = w & np.uint64(0xFFFF), w >> np.uint64(16)
    return out.reshape(rows, blocks * 8)[:, :width]


def keep_mask(p: float, seed: int, offset: int, rows: int, width: int) -> torch.Tensor:
    """0 or 65536 / kept, in 64 bits."""
    kept = round((1 - p) * 65536)
    return torch.from_numpy(np.where(lanes(seed, offset, rows, width) < kept, 65536 / max(kept, 1), 0.0))


# ------------------------------------------------------------------------------------------
# Block norm: rows [rows, width] of doubles; gate [groups, width] with gate_rows rows each
# ------------------------------------------------------------------------------------------
def spread_gate(gate, gate_rows, rows):
    return gate.repeat_interleave(gate_rows, 0)[:rows] if gate is not None else 1.0


def block_norm(x, b, w_post, gate, gate_rows, w_next, alpha, beta, w0, eps, mask):
    """(h, its magnitude, a, its magnitude, r, s)."""
    r = s = a = a_mag = None
    h, mag = alpha * x, abs(alpha) * x.abs()
    if b is not None:
        n = b
        if w_post is not None:
            r = (b.square().mean(1) + eps).rsqrt()
            n = b * r[:, None] * (w0 + w_post)
        n = beta * mask * spread_gate(gate, gate_rows, len(x)) * n
        h, mag = h + n, mag + n.abs()
    if w_next is not None:
        s = (h.square().mean(1) + eps).rsqrt()
        a = h * s[:, None] * (w0 + w_next)
        # an error e of h moves a by s |w| |e|, and through s by at most |a| times e's share of the row
        share = (mag.square().mean(1).sqrt() * s)[:, None]
        a_mag = (mag * s[:, None] + share * h.abs() * s[:, None]) * (w0 + w_next).abs()
    return h, mag, a, a_mag, r, s


def block_norm_backward(dh, da, h, b, r, s, w_post, gate, gate_rows, w_next, alpha, beta, w0, mask):
    """{name: (gradient, its magnitude)}, from the stored h, r and s."""
    out = {}
    H = dh if dh is not None else torch.zeros_like(h)
    mag = H.abs()
    if w_next is not None:
        s = s[:, None]
        p = da * (w0 + w_next)
        H = H + s * p - h * s ** 3 * (p * h).mean(1, keepdim=True)
        mag = mag + s * p.abs() + h.abs() * s ** 3 * (p * h).abs().mean(1, keepdim=True)
        out["next_weight"] = (da * h * s).sum(0), (da * h * s).abs().sum(0)
    out["residual"] = alpha * H, abs(alpha) * mag
    if b is not None:
        g = spread_gate(gate, gate_rows, len(h))
        ga = g.abs() if gate is not None else 1.0
        t, t_mag = beta * mask * H, abs(beta) * mask * mag
        unit = b * r[:, None] if w_post is not None else b
        w = (w0 + w_post) if w_post is not None else torch.ones(h.shape[1], dtype=torch.float64)
        u, u_mag = t * g * w, t_mag * ga * w.abs()
        if w_post is not None:
            r = r[:, None]
            out["branch"] = (r * u - b * r ** 3 * (u * b).mean(1, keepdim=True),
                             r * u_mag + b.abs() * r ** 3 * (u_mag * b.abs()).mean(1, keepdim=True))
            out["post_weight"] = (t * g * unit).sum(0), (t_mag * ga * unit.abs()).sum(0)
        else:
            out["branch"] = u, u_mag
        if gate is not None:
            def groups(v):
                pad = len(gate) * gate_rows - len(v)
                return torch.cat([v, v.new_zeros(pad, v.shape[1])]).view(len(gate), gate_rows, -1).sum(1)

            out["gate"] = groups(t * unit * w), groups(t_mag * unit.abs() * w.abs())
    return out


# ------------------------------------------------------------------------------------------
# Rotary: x [batch, length, heads, head_dim] of doubles, positions [batch, length]
# ------------------------------------------------------------------------------------------
def rotary(x, positions, frequencies, scale, interleaved, inverse):
    """(result, magnitude)."""
    t = positions.double()[:, :, None] * frequencies
    c, s = torch.cos(t)[:, :, None] * scale, torch.sin(t)[:, :, None] * (-scale if inverse else scale)
    half = len(frequencies)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    mag[..., a] = mag[..., b] = (x[..., a].abs() + x[..., b].abs()) * abs(scale)
    return y, mag


# ------------------------------------------------------------------------------------------
# Logits: a row at a time, a token at a time where the lists are concerned
# ------------------------------------------------------------------------------------------
def logits_rules(x, tokens=None, lengths=None, prompt_lengths=None, repetition=None, frequency=None, presence=None,
                 bias_tokens=None, bias_values=None, mask=None):
    """(result, magnitude) of doubles [rows, vocab]; lists are Python lists for each row."""
    y, mag = x.clone(), x.abs()
    vocab = x.shape[1]
    for i in range(len(x)):
        if tokens is not None:
            row = tokens[i]
            row = row[:min(len(row), max(0, lengths[i]))] if lengths is not None else row
            prompt = max(0, prompt_lengths[i]) if prompt_lengths is not None else 0
            for v in {v for v in row if 0 <= v < vocab}:
                count = sum(1 for j, t in enumerate(row) if t == v and j >= prompt)
                l = y[i, v].item()
                if repetition is not None:
                    l = (l / repetition[i] if repetition[i] else math.copysign(math.inf, l)) if l > 0 else l * repetition[i]
                m = abs(l)
                if frequency is not None:
                    l, m = l - frequency[i] * count, m + abs(frequency[i]) * count
                if presence is not None and count:
                    l, m = l - presence[i], m + abs(presence[i])
                y[i, v], mag[i, v] = l, m
        if bias_tokens is not None:
            for v, value in dict(zip(bias_tokens[i], bias_values[i])).items():
                if 0 <= v < vocab:
                    y[i, v] += value
                    mag[i, v] += abs(value)
        if mask is not None:
            for v in range(vocab):
                if not mask[i][v // 32] >> (v % 32) & 1:
                    y[i, v] = -math.inf
    return y, torch.where(torch.isfinite(mag), mag, 0.0)
