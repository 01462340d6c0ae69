"""Plain implementations of the attention operators in 64 bits, on the CPU, and the bounds that the kernels' results are
held to.

Bounds of attention.  u = 2^-24; a product sum of D terms in 32 bits, whatever its order and with a tensor core's
truncating additions (2^-23 each), is off by at most (D + 4) 2^-23 of the sum of magnitudes, so a score (in natural units) by
    d = (D + 4) 2^-23 scale max_j sum |q k_j|
plus what the scaling to base 2 and the subtraction of the maximum round, 2^-22 of the largest score's magnitude.  A weight is
off by that and by the exponential's own error e (2^-21 in 32 bits; 2^-12 where half types take a polynomial), and, for half
types, rounded to 16 bits before it meets a value (bfloat16 2^-8, float16 2^-11).  Numerator and denominator are sums of n
weights.  So
    |got - exact| <= 2^-p |exact| + (2 d + 2 e + r + 2 n 2^-23) sum_j p_j |v_j|
with r the rounding of the weights (0 for float32) and 2^-p the rounding of the result.
"""
from __future__ import annotations

import torch

from tests.lm_reference import ROUND, TINY


def score_error(head: int, magnitude: torch.Tensor) -> torch.Tensor:
    """magnitude: scale times the largest sum of |q k| of a row."""
    return (head + 4) * 2.0 ** -23 * magnitude + 2.0 ** -22 * magnitude


def attend(q, k, v, scale, seen, dtype):
    """Rows q [n, d] over keys k, v [m, d] where seen [n, m] (64 bits): (result, bound of a result stored in dtype)."""
    d, m = q.shape[1], k.shape[0]
    if m == 0:
        zero = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
        return zero, zero
    scores = (q @ k.T * scale).masked_fill(~seen, -torch.inf)
    any_seen = seen.any(1, keepdim=True)
    p = torch.where(any_seen, scores.softmax(1), 0.0).masked_fill(~seen, 0.0)
    magnitude = (q.abs() @ k.abs().T * abs(scale)).masked_fill(~seen, 0.0).amax(1, keepdim=True)
    error = score_error(d, magnitude)
    half = dtype != torch.float32
    rounding = (ROUND[dtype] if half else 0.0) + 2 * (2.0 ** -12 if half else 2.0 ** -21) + 2 * m * 2.0 ** -23
    # a value that is not seen may be anything
    o = torch.stack([p[i][seen[i]] @ v[seen[i]] for i in range(len(q))]) if not torch.isfinite(v).all() else p @ v
    mag = torch.stack([p[i][seen[i]] @ v[seen[i]].abs() for i in range(len(q))]) if not torch.isfinite(v).all() else p @ v.abs()
    return o, ROUND[dtype] * o.abs() + (2 * error + rounding) * mag + TINY[dtype]


def assert_close(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str = "") -> None:
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} != {tuple(want.shape)}"
    g = got.detach().cpu().double()
    bad = ~((g - want).abs() <= bound) & ~((g == want) | (torch.isnan(g) & torch.isnan(want)))
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {g.numel()} outside the bound; first {i}: got {g[i].item()!r}, "
                             f"exact {want[i].item()!r}, bound {bound[i].item()!r}")


def prompt(q, k, v, starts, k_starts, scale, causal, dtype, out=None):
    """(result, bound) [tokens, heads, d] of doubles; rows of no sequence as in out, or 0."""
    want = torch.zeros(q.shape, dtype=torch.float64) if out is None else out.clone()
    bound = torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[1] // k.shape[1]
    for a, b, ka, kb in zip(starts, starts[1:], k_starts, k_starts[1:]):
        n, m = b - a, kb - ka
        seen = torch.ones(n, m, dtype=torch.bool)
        if causal:
            seen = torch.arange(m) <= torch.arange(n)[:, None] + (m - n)
        for h in range(q.shape[1]):
            if n:
                want[a:b, h], bound[a:b, h] = attend(q[a:b, h], k[ka:kb, h // group], v[ka:kb, h // group], scale, seen, dtype)
    return want, bound


def decode(q, k, v, table, lengths, scale, dtype):
    """q [batch, heads, d]; k, v [pages, page_size, heads, d] of doubles: (result, bound)."""
    want, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    pages, page = k.shape[:2]
    group = q.shape[1] // k.shape[2]
    for b in range(len(q)):
        at = torch.arange(max(0, min(int(lengths[b]), table.shape[1] * page)))
        index = table[b].long()[at // page]
        ok = (index >= 0) & (index < pages)
        kb, vb = k[index[ok], at[ok] % page], v[index[ok], at[ok] % page]
        for h in range(q.shape[1]):
            seen = torch.ones(1, len(kb), dtype=torch.bool)
            w, e = attend(q[b, h:h + 1], kb[:, h // group], vb[:, h // group], scale, seen, dtype)
            want[b, h], bound[b, h] = w[0], e[0]
    return want, bound


def e4m3(y: torch.Tensor) -> torch.Tensor:
    """Doubles rounded to nearest even to 4 significant bits, multiples of 2^-9 below 2^-6, at most 448."""
    _, e = torch.frexp(y.abs().clamp(min=2.0 ** -6))
    step = torch.exp2((e - 4).double())
    return (torch.round(y / step) * step).clamp(-448, 448)


def quantise(x: torch.Tensor):
    """Rows of doubles: (what the cache's 8 bits stand for, exponents)."""
    finite = torch.where(torch.isfinite(x), x, 0.0)
    top, e = torch.frexp(finite.abs().amax(-1))
    e = torch.where(top > 0, e - 9 + (top > 0.875), 0).clamp(-96, 96)
    scale = torch.exp2(e.double())[..., None]
    return torch.where(torch.isfinite(x), e4m3(finite / scale) * scale, torch.nan), e


def head_norm(x, w, w0, eps, positions, f, scale, interleaved):
    """x [batch, length, heads, d] of doubles: (result, magnitude, rstd)."""
    r = (x.square().mean(-1) + eps).rsqrt()
    n = x * r[..., None] * (w0 + w if w is not None else 1.0)
    y, mag = n.clone(), n.abs()
    a, b = pairs(len(f), interleaved)
    t = positions.double()[:, :, None] * f
    c, s = torch.cos(t)[:, :, None] * scale, torch.sin(t)[:, :, None] * scale
    y[..., a], y[..., b] = n[..., a] * c - n[..., b] * s, n[..., a] * s + n[..., b] * c
    mag[..., a] = mag[..., b] = (n[..., a].abs() + n[..., b].abs()) * abs(scale)
    return y, mag, r


def pairs(half, interleaved):
    return (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))


def head_norm_backward(dy, x, w, w0, r, positions, f, scale, interleaved):
    """{name: (gradient, magnitude)} of x and the weight, from the saved r."""
    a, b = pairs(len(f), interleaved)
    t = positions.double()[:, :, None] * f
    c, s = torch.cos(t)[:, :, None] * scale, torch.sin(t)[:, :, None] * scale
    g, g_mag = dy.clone(), dy.abs()
    g[..., a], g[..., b] = dy[..., a] * c + dy[..., b] * s, dy[..., b] * c - dy[..., a] * s
    g_mag[..., a] = g_mag[..., b] = (dy[..., a].abs() + dy[..., b].abs()) * abs(scale)
    wp = w0 + w if w is not None else torch.ones(x.shape[-1], dtype=torch.float64)
    r = r[..., None]
    e, u, u_mag = x * r, g * wp, g_mag * wp.abs()
    dx = r * (u - e * (u * e).mean(-1, keepdim=True))
    mag = r * (u_mag + e.abs() * (u_mag * e.abs()).mean(-1, keepdim=True))
    return {"x": (dx, mag), "weight": ((g * e).sum((0, 1, 2)), (g_mag * e.abs()).sum((0, 1, 2)))}
