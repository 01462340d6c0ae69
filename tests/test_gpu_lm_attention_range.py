"""Attention whose weights, scales and queries span a wide range: what contributes least to the maximum, or beside it, has to
reach the output all the same (mtxc_decode_attention, mtxc_prompt_attention, against the formulas in 64 bits).

Bounds, for a row whose exact weights are p_j, with the terms that attention_reference derives for scores (d), exponentials (e),
the rounding of weights to 16 bits (r) and of the result.  Sums: a product of 16 keys adds to a sum in 32 bits once, a truncation
of 2^-23, so m keys take m / 16 of them (m in the kernels for any head) and 16 for their own sum and the joins.  float16 weights
are multiples of 2^-24, 2^15 (prompts: 2^11) for the largest one or more: off by another 2^-25 / 2^15 of it, whatever their size.
Over 8 bits a weight carries its value's scale a_j = 2^exponent, and stands beside v_j / a_j:
    |got - exact| <= 2^-p |exact| + (2 d + 2 e + r + 2 (m / 16 + 16) 2^-23) sum_j p_j |v_j|
                     + 2^-40 max_j(p_j a_j) sum_j |v_j| / a_j
(a_j = 1 elsewhere; 2^-36 in prompts; no such term for other types), and exponents of up to E beside scores in powers of two
round by 2^-22 E more in d.
"""
import math

import pytest
import torch

from tests import attention_reference as att
from tests.lm_reference import ROUND, TINY

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
KINDS = [(t, k) for t in (torch.float32, torch.float16, torch.bfloat16) for k in (t, E4M3)]
HALVES = [(t, k) for t, k in KINDS if t != torch.float32]


@pytest.fixture
def lm(gpu):
    from matrix_b200 import lm

    return lm


def attend(q, k, v, scale, dtype, kind, exponents=None, step=2.0 ** -40, seen=None):
    """Rows q [n, d] over k, v [m, d] (64 bits; seen [n, m]): (result, bound)."""
    m = k.shape[0]
    seen = torch.ones(len(q), m, dtype=torch.bool) if seen is None else seen
    p = (q @ k.T * scale).masked_fill(~seen, -torch.inf).softmax(1)
    o, mag = p @ v, p @ v.abs()
    half = dtype != torch.float32
    weights = torch.float32 if not half else torch.float16 if kind == E4M3 else kind
    d = att.score_error(q.shape[1], (q.abs() @ k.abs().T * abs(scale)).masked_fill(~seen, 0.0).amax(1, keepdim=True))
    a = torch.ones(m, dtype=torch.float64) if exponents is None else torch.exp2(exponents.double())
    if exponents is not None:
        d = d + 2.0 ** -22 * exponents.abs().max()
    work = 2 * d + 2 * (2.0 ** -12 if half else 2.0 ** -21) + (ROUND[weights] if half else 0.0)
    work = work + 2 * ((m / 16 if half else m) + 16) * 2.0 ** -23
    floor = step * (p * a).amax(1, keepdim=True) * (seen.double() @ (v.abs() / a[:, None])) if weights == torch.float16 else 0.0
    return o, ROUND[dtype] * o.abs() + work * mag + floor + TINY[dtype]


def stored(lm, k, v, kind, page=64):
    """A cache of one head that holds k, v [n, d] (in 8 bits: bytes of their own, with exponents 0), and its page table."""
    n, head = k.shape
    pages = (n + page - 1) // page
    cache = lm.kv_cache(pages, page, 1, head, kind)
    at = torch.randperm(pages, generator=torch.Generator().manual_seed(n))
    slots = at[torch.arange(n) // page] * page + torch.arange(n) % page
    for x, to in ((k, cache.keys), (v, cache.values)):
        to.view(torch.int8 if kind == E4M3 else kind)[slots // page, slots % page, 0] = \
            x.to(kind).view(torch.int8 if kind == E4M3 else kind).cuda()
    return cache, at.to(torch.int32)[None].cuda(), slots


def decode(lm, q, cache, table, n, scale):
    return lm.decode_attention(q[None].cuda(), cache, table, torch.tensor([n], dtype=torch.int32).cuda(), scale=scale)[0]


def check_decode(lm, q, cache, table, n, scale, want, bound, what=""):
    """As one sequence, whose tiles workers share, and as many, of which a worker has several tiles and whole sequences."""
    att.assert_close(decode(lm, q, cache, table, n, scale), want, bound, what)
    many = 1 + 500000 // n
    lengths = torch.full((many,), n, dtype=torch.int32).cuda()
    got = lm.decode_attention(q[None].expand(many, -1, -1).cuda(), cache, table.expand(many, -1), lengths, scale=scale)
    different = (got - got[0]).abs().flatten(1).amax(1).nonzero()[:, 0].tolist()
    for i in [0, *different[:20], many - 1]:
        att.assert_close(got[i], want, bound, f"{what}, {i} of {many}")
    low, high = got.amin(0), got.amax(0)
    att.assert_close(low, want, bound, what)
    att.assert_close(high, want, bound, what)


def powers(bits, head):
    """The scale with which rows of ones have 2^bits times the weight of zeros."""
    return bits * math.log(2.0) / head


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("top", [1e-3, 1e-5, 1e-20])
@pytest.mark.parametrize("head,heads", [(64, 4), (128, 12)])
def test_decode_zero_rows_beside_small_ones(lm, dtype, top, head, heads):
    """Values of zeros, whose scale in 8 bits is 2^0, count for the denominator alone, wherever they lie."""
    if dtype == torch.float16 and top < 1e-5:
        pytest.skip("no float16 of this size")
    page = 16
    g = torch.Generator().manual_seed(head)
    for n, zeros in ((900, slice(0, 300)), (900, slice(600, 900)), (900, slice(1, None, 2)), (900, slice(0, 899)), (900, slice(None)),
                     (200, slice(0, 70)), (200, slice(100, 200)), (200, slice(1, None, 2)), (20, slice(0, 19))):
        k, v = torch.randn(n, 1, head, generator=g), torch.randn(n, 1, head, generator=g) * top
        v[zeros] = 0.0
        k, v, q = k.to(dtype), v.to(torch.bfloat16).float(), torch.randn(heads, head, generator=g).to(dtype)
        cache = lm.kv_cache(60, page, 1, head, E4M3)
        table = torch.arange((n + page - 1) // page, dtype=torch.int32)[None].cuda()
        slots = torch.arange(n).cuda()
        lm.cache_write(cache, k.float().cuda(), v.cuda(), slots)
        (k, _), (v, e) = att.quantise(k[:, 0].double()), att.quantise(v[:, 0].double())
        e = torch.where(v.any(1), e, -96)  # a row of zeros has no say in the weights' step
        want, bound = attend(q.double(), k, v, head ** -0.5, dtype, E4M3, e.long())
        check_decode(lm, q, cache, table, n, None, want, bound, f"{dtype} {top} {zeros}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [40, 3000])
def test_decode_scales_at_the_ends(lm, dtype, n):
    """Keys of nearly all the weight whose values' scales are 2^-90, others with 2^90: the values of the others are the output,
    the weights of the first the denominator."""
    head = 64
    g = torch.Generator().manual_seed(n)
    for bits in (30, 100):
        for order in (slice(0, n // 2), slice(n // 2, n), slice(0, None, 2)):
            k, e = torch.zeros(n, head), torch.full((n,), 90)
            k[order], e[order] = 1.0, -90
            v = (torch.rand(n, head, generator=g) * 200 + 200).to(E4M3).double()
            cache, table, slots = stored(lm, k, v, E4M3)
            cache.value_exponents[slots // 64, slots % 64, 0] = e.to(torch.int8).cuda()
            v = v * torch.exp2(e.double())[:, None]
            q = torch.ones(4, head, dtype=dtype)
            want, bound = attend(q.double(), k.double(), v, powers(bits, head), dtype, E4M3, e)
            check_decode(lm, q, cache, table, n, powers(bits, head), want, bound, f"{bits} {order}")


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("bits", [16.3, 22.4, 24.8, 25.2])
@pytest.mark.parametrize("n,heads,head", [(2500, 4, 64), (2500, 16, 128), (40000, 4, 64)])
def test_decode_one_key_far_above_the_others(lm, dtype, kind, bits, n, heads, head):
    """A key with nearly all the weight and zeros but for one element as its value: the rest of the output is what the others
    are worth together, each of a weight 2^-bits."""
    g = torch.Generator().manual_seed(n + heads)
    for where in (0, n // 2, n - 1):
        k = torch.zeros(n, head)
        k[where] = 1.0
        v = (torch.rand(n, head, generator=g) * 100 + 100).to(kind).float()
        v[where, 1:] = 0.0
        cache, table, _ = stored(lm, k, v, kind)
        q = torch.ones(heads, head, dtype=dtype)
        scale = powers(bits, head)
        want, bound = attend(q.double(), k.double(), v.double(), scale, dtype, kind)
        check_decode(lm, q, cache, table, n, scale, want, bound, f"{dtype} {kind} {where}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [3.9, 7.9, 16.3, 22.4, 24.8])
@pytest.mark.parametrize("head", [64, 128, 256])
def test_prompt_one_key_far_above_the_others(lm, dtype, bits, head):
    """The same in a prompt, with the key in the first tile of keys or a later one."""
    n, scale = 1500, powers(bits, head)
    g = torch.Generator().manual_seed(head)
    for where in (0, 400):
        q, k = torch.ones(n, 2, head, dtype=dtype), torch.zeros(n, 1, head, dtype=dtype)
        k[where] = 1.0
        v = (torch.rand(n, 1, head, generator=g) * 100 + 100).to(dtype)
        v[where, :, 1:] = 0.0
        got = lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), scale=scale)
        seen = torch.ones(n, n, dtype=torch.bool).tril()
        want, bound = attend(q[:, 0].double(), k[:, 0].double(), v[:, 0].double(), scale, dtype, dtype, None, 2.0 ** -36, seen)
        for h in range(2):
            att.assert_close(got[:, h], want, bound, f"{dtype} {where}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,head", [(4, 64), (12, 128)])
def test_decode_queries_with_one_large_element_over_8_bits(lm, dtype, heads, head):
    """A query's element of 2^12 against zeros in the keys, the others of 2^-9: those make the scores."""
    n = 500
    g = torch.Generator().manual_seed(head)
    k, v = ((torch.randn(n, head, generator=g) * 2).to(E4M3).float() for _ in range(2))
    k[:, 3] = 0.0
    q = (torch.randn(heads, head, generator=g) * 2.0 ** -9).to(dtype)
    q[:, 3] = 2.0 ** 12
    cache, table, _ = stored(lm, k, v, E4M3)
    scale = 512 / head ** 0.5
    want, bound = attend(q.double(), k.double(), v.double(), scale, dtype, E4M3)
    check_decode(lm, q, cache, table, n, scale, want, bound)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,head", [(4, 64), (16, 128), (12, 200), (3, 66)])
def test_decode_weights_keep_more_than_16_bits(lm, dtype, heads, head):
    """Values of two keys that would cancel if the weight of one, 2^-1 and 0.4 steps of its type, were rounded to it.  The weights are
    kept as two parts of 16 bits, so r is the square of the type's rounding, and the exponentials are those of 32 bits."""
    n, weight = 120, 0.5 + 0.4 * ROUND[dtype]
    k, v = torch.zeros(n, head), torch.ones(n, head)
    k[1::2], v[1::2] = -1.0, -2.0
    cache, table, _ = stored(lm, k, v, dtype)
    q, scale = torch.ones(heads, head, dtype=dtype), -math.log(weight) / head
    p = (q.double() @ k.double().T * scale).softmax(1)
    want, mag = p @ v.double(), p @ v.abs().double()
    d = att.score_error(head, torch.full((heads, 1), -math.log(weight), dtype=torch.float64))
    work = 2 * d + 2 * 2.0 ** -21 + ROUND[dtype] ** 2 + 2 * (n + 16) * 2.0 ** -24
    bound = ROUND[dtype] * want.abs() + work * mag + 2.0 ** -40 * p.amax() * n + TINY[dtype]
    assert (want.abs() > 2 * bound).all()
    check_decode(lm, q, cache, table, n, scale, want, bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,head", [(4, 64), (16, 128), (3, 66)])
def test_decode_infinite_values_that_are_seen(lm, dtype, heads, head):
    """An infinity among the values is the output's in its element, against a weight of 1, of a power of two and of neither; of both
    signs, or with NaN, it is NaN."""
    n = 90
    g = torch.Generator().manual_seed(head)
    k, v = torch.zeros(n, head), torch.randn(n, head, generator=g).to(dtype).float()
    k[10:20], k[20:30] = -1.0, -1.3
    inf = float("inf")
    want_of = {1: (0, inf), 2: (15, inf), 3: (25, -inf), 4: (89, -inf), 5: (40, float("nan"))}
    for c, (at, x) in want_of.items():
        v[at, c] = x
    v[3, 6], v[70, 6] = inf, -inf
    cache, table, _ = stored(lm, k, v, dtype)
    for scale in (math.log(2.0) / head, 9 * math.log(2.0) / head):  # 1/2 and 2^-1.3, 2^-9 and 2^-11.7
        got = decode(lm, torch.ones(heads, head, dtype=dtype), cache, table, n, scale).float().cpu()
        for c, (_, x) in want_of.items():
            assert (got[:, c] == x).all() if x == x else torch.isnan(got[:, c]).all(), (c, got[:, c])
        assert torch.isnan(got[:, 6]).all() and torch.isfinite(got[:, 7:]).all() and torch.isfinite(got[:, 0]).all()
