"""Attention of one token over a paged cache and of whole prompts (mtxc_decode_attention, mtxc_prompt_attention) against the
formulas in 64 bits, within the bounds that attention_reference derives."""
import threading

import pytest
import torch

from tests import attention_reference as att

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
E4M3 = torch.float8_e4m3fn
KEPT = []


@pytest.fixture
def lm(gpu):
    from matrix_b200 import lm

    return lm


def normal(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed * 31 + sum(shape))
    return (torch.randn(*shape, generator=g) * std).to(dtype)


# ------------------------------------------------------------------------------------------
# One token
# ------------------------------------------------------------------------------------------
def filled(lm, pages, page, heads, head, kind, seed=0, std=1.0):
    """A cache on the device and what it holds, in 64 bits."""
    cache = lm.kv_cache(pages, page, heads, head, kind)
    shape = (pages, page, heads, head)
    held = []
    for i, (x, e) in enumerate(((cache.keys, cache.key_exponents), (cache.values, cache.value_exponents))):
        y = normal(*shape, seed=seed + i, std=std)
        if kind == E4M3:
            g = torch.Generator().manual_seed(seed + i)
            exponents = torch.randint(-9, -3, shape[:3], generator=g)
            y = (y * 100).clamp(-448, 448).to(E4M3)
            x.copy_(y.cuda())
            e.copy_(exponents.cuda())
            held.append(y.double() * torch.exp2(exponents.double())[..., None])
        else:
            x.copy_(y.to(kind).cuda())
            held.append(y.to(kind).double())
    return cache, *held


def tables(lengths, page, pages, seed=0, width=None):
    used = [(max(0, n) + page - 1) // page for n in lengths]
    width = max(1, *used) if width is None else width
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    g = torch.Generator().manual_seed(seed)
    for i, n in enumerate(used):
        table[i, :n] = torch.randint(0, pages, (n,), generator=g)  # sequences may share pages
    return table


def check_decode(lm, dtype, kind, lengths, qh, kh, head, page, pages=12, scale=None, seed=0, std=1.0, **more):
    cache, k, v = filled(lm, pages, page, kh, head, kind, seed, std)
    q = normal(len(lengths), qh, head, dtype=dtype, seed=seed + 5)
    table = tables(lengths, page, pages, seed)
    n = torch.tensor(lengths, dtype=torch.int32)
    got = lm.decode_attention(q.cuda(), cache, table.cuda(), n.cuda(), scale=scale, **more)
    s = head ** -0.5 if scale is None else scale
    want, bound = att.decode(q.double(), k, v, table, lengths, s, dtype)
    att.assert_close(got, want, bound, f"{dtype} {kind} {lengths} {qh}/{kh} x {head} page {page}")
    return got


KINDS = [(t, k) for t in TYPES for k in (t, E4M3)]


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("head", [1, 3, 8, 16, 40, 64, 66, 80, 96, 112, 128, 136, 192, 200, 256])
def test_decode_heads(lm, dtype, kind, head):
    check_decode(lm, dtype, kind, [1, 37, 0, 130], 4, 2, head, 16)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("qh,kh", [(1, 1), (3, 3), (7, 1), (8, 1), (14, 2), (16, 1), (17, 1), (32, 2), (40, 1), (64, 8)])
def test_decode_groups(lm, dtype, kind, qh, kh):
    check_decode(lm, dtype, kind, [65, 300], qh, kh, 64, 16)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("page", [1, 2, 7, 16, 24, 64, 100, 128])
@pytest.mark.parametrize("head", [64, 128])
def test_decode_pages(lm, dtype, kind, page, head):
    """Pages that end inside a tile, and lengths around their borders."""
    lengths = [1, max(1, page - 1), page, page + 1, 2 * page + 1, 31, 32, 33, 127, 128, 129]
    check_decode(lm, dtype, kind, lengths, 8, 2, head, page, pages=20)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("lengths", [[5000], [1] * 300, [3000, 1, 0, 0, 700, 2500], [0], [0, 0, 9], list(range(0, 200, 3))])
def test_decode_lengths(lm, dtype, kind, lengths):
    """One long sequence that many blocks share, many short ones, empty ones in between."""
    check_decode(lm, dtype, kind, lengths, 8, 2, 64, 16, pages=64)


@pytest.mark.parametrize("dtype,kind", KINDS)
def test_decode_peaked_scores(lm, dtype, kind):
    """Scores of magnitude 50 and more: one key has nearly all the weight, and the maximum moves along the cache."""
    check_decode(lm, dtype, kind, [900, 300], 4, 2, 64, 16, pages=40, scale=3.0, std=2.0)
    check_decode(lm, dtype, kind, [900, 300], 4, 2, 64, 16, pages=40, scale=-1.0)
    check_decode(lm, dtype, kind, [900, 300], 4, 2, 64, 16, pages=40, scale=0.0)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("head", [64, 66])
def test_decode_ignores_what_lies_behind_a_length(lm, dtype, kind, head):
    """NaN and infinities in the slots behind the lengths, in pages of other sequences, and pages that do not exist."""
    page, pages = 16, 8
    cache, k, v = filled(lm, pages, page, 2, head, kind)
    q = normal(3, 4, head, dtype=dtype)
    table = torch.tensor([[0, 1, 6, 6], [2, 3, 4, 7], [5, 6, -5, 1 << 30]], dtype=torch.int32)
    lengths = [20, 50, 16]
    bad = torch.zeros(pages, page, dtype=torch.bool)
    bad[1, 4:], bad[4, 2:], bad[6], bad[7, 2:] = True, False, True, True
    for x in (cache.keys, cache.values):
        if kind == E4M3:
            x.view(torch.int8)[bad.cuda()] = 0x7F
        else:
            x[bad.cuda()] = float("nan")
            x[1, 5:] = float("inf")
    got = lm.decode_attention(q.cuda(), cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
    want, bound = att.decode(q.double(), k, v, table, lengths, head ** -0.5, dtype)
    assert torch.isfinite(want).all()
    att.assert_close(got, want, bound)


@pytest.mark.parametrize("dtype,kind", KINDS)
def test_decode_bad_pages_and_lengths(lm, dtype, kind):
    """Tokens in pages that the cache does not have are passed over; lengths past the table are cut to it, negative ones
    are empty; nothing left gives 0."""
    cache, k, v = filled(lm, 6, 16, 2, 64, kind)
    q = normal(5, 8, 64, dtype=dtype)
    table = torch.tensor([[0, -1, 2], [6, 1, 1 << 30], [-7, 99, 6], [3, 4, 5], [1, 1, 1]], dtype=torch.int32)
    lengths = [48, 40, 48, 1 << 30, -4]
    got = lm.decode_attention(q.cuda(), cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
    want, bound = att.decode(q.double(), k, v, table, lengths, 0.125, dtype)
    att.assert_close(got, want, bound)
    assert not got[2].any() and not got[4].any()


@pytest.mark.parametrize("dtype,kind", [(t, t) for t in TYPES])
def test_decode_infinite_and_nan_scores(lm, dtype, kind):
    """A key with an infinity against it gets no weight; one with NaN makes its rows NaN, and no others."""
    cache, k, v = filled(lm, 6, 16, 2, 64, kind)
    q = normal(2, 4, 64, dtype=dtype).abs() + 0.125
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
    cache.keys[0, 3, 0, 7] = -float("inf")
    cache.keys[4, 3, 1, 7] = float("nan")
    lengths = [40, 48]
    got = lm.decode_attention(q.cuda(), cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()).cpu()
    want, bound = att.decode(q.double(), k, v, table, lengths, 0.125, dtype)
    rows = k[:3].flatten(0, 1)[:40, 0], v[:3].flatten(0, 1)[:40, 0]
    want[0, :2], bound[0, :2] = att.attend(q[0, :2].double(), *rows, 0.125, (torch.arange(40) != 3).expand(2, 40), dtype)
    want[1, 2:] = torch.nan
    att.assert_close(got, want, bound)


def test_decode_scales_of_8_bits_far_apart(lm):
    """Values whose scales differ by 2^40, the largest at keys of small weight and the other way round; keys likewise."""
    page, pages, head = 16, 6, 64
    for dtype in TYPES:
        for turn in (0, 1):
            cache, k, v = filled(lm, pages, page, 1, head, E4M3)
            e = torch.zeros(pages, page, 1, dtype=torch.int64)
            e[::2] = 20 if turn else -20
            e[1::2] = -20 if turn else 20
            cache.value_exponents.copy_(e.cuda())
            v = cache.values.cpu().double() * torch.exp2(e.double())[..., None]
            f = torch.full((pages, page, 1), -40, dtype=torch.int64)
            f[2:4] = -7
            cache.key_exponents.copy_(f.cuda())
            k = cache.keys.cpu().double() * torch.exp2(f.double())[..., None]
            q = normal(1, 3, head, dtype=torch.float32, std=8.0).to(dtype)
            table = torch.arange(pages, dtype=torch.int32)[None]
            got = lm.decode_attention(q.cuda(), cache, table.cuda(), torch.tensor([90], dtype=torch.int32).cuda())
            want, bound = att.decode(q.double(), k, v, table, [90], head ** -0.5, dtype)
            if dtype == torch.float16:  # what passes its largest is stored as an infinity
                over = want.abs() > 65504 * (1 - 2.0 ** -8)
                want, bound, got = want[~over], bound[~over], got.cpu()[~over]
            att.assert_close(got, want, bound, f"{dtype} {turn}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [2.0 ** -100, 1.0, 2.0 ** 60])
def test_decode_queries_of_any_size_over_8_bits(lm, dtype, scale):
    if dtype == torch.float16:
        scale = {2.0 ** -100: 2.0 ** -12, 1.0: 1.0, 2.0 ** 60: 2.0 ** 12}[scale]
    cache, k, v = filled(lm, 6, 16, 2, 64, E4M3)
    q = (normal(2, 4, 64) * scale).to(dtype)
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
    got = lm.decode_attention(q.cuda(), cache, table.cuda(), torch.tensor([40, 48], dtype=torch.int32).cuda(), scale=0.125 / scale)
    want, bound = att.decode(q.double(), k, v, table, [40, 48], 0.125 / scale, dtype)
    att.assert_close(got, want, bound)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("head", [64, 128, 60])
def test_decode_layouts(lm, dtype, kind, head):
    """Slots before heads, caches and queries that are parts of larger tensors, misaligned; outputs that are given, the
    queries themselves among them; a table with a stride."""
    lengths, page, pages = [70, 33], 16, 8
    cache, k, v = filled(lm, pages, page, 2, head, kind)
    plain = lm.KVCache(*(t.contiguous() if t is not None else None for t in cache))
    # parts of larger tensors, one element further
    wide = [torch.zeros(pages, page, 3, head + 9, dtype=torch.int8 if kind == E4M3 else kind, device="cuda").view(kind) for _ in range(2)]
    for w, t in zip(wide, cache[:2]):
        w[:, :, 1:, 1:head + 1].copy_(t)
    shifted = lm.KVCache(*(w[:, :, 1:, 1:head + 1] for w in wide), *cache[2:])
    table = tables(lengths, page, pages)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    big = normal(2, 9, head + 3, dtype=dtype).cuda()
    q = big[:, 2:8, 1:head + 1]
    spread = torch.stack([table, table * 0], 0).cuda()[0]
    want, bound = att.decode(q.cpu().double(), k, v, table, lengths, head ** -0.5, dtype)
    for c in (cache, plain, shifted):
        att.assert_close(lm.decode_attention(q, c, spread, n), want, bound)
        att.assert_close(lm.decode_attention(q.contiguous(), c, table.cuda(), n), want, bound)
    before, version = big.clone(), big._version
    got = lm.decode_attention(q, cache, table.cuda(), n, out=q)
    assert got is q and big._version > version
    att.assert_close(q, want, bound)
    before[:, 2:8, 1:head + 1] = q
    assert torch.equal(before, big)


def test_decode_a_cache_past_32_bits(lm):
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("not enough memory")
    pages, page, heads, head = 40, 16, 2, 128
    stride = (1 << 32) // 36 // 128 * 128
    cache = []
    for i in range(2):
        base = torch.empty(pages * stride, dtype=torch.bfloat16, device="cuda")
        t = torch.as_strided(base, (pages, page, heads, head), (stride, heads * head, head, 1))
        t.copy_(normal(pages, page, heads, head, seed=i))
        cache.append(t)
    q = normal(2, 4, head, dtype=torch.bfloat16)
    table = torch.tensor([[39, 38, 37], [1, 39, 20]], dtype=torch.int32)
    got = lm.decode_attention(q.cuda(), lm.KVCache(*cache), table.cuda(), torch.tensor([48, 40], dtype=torch.int32).cuda())
    want, bound = att.decode(q.double(), cache[0].cpu().double(), cache[1].cpu().double(), table, [48, 40], head ** -0.5, torch.bfloat16)
    att.assert_close(got, want, bound)


@pytest.mark.parametrize("dtype,kind", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, E4M3)])
def test_decode_recorded_on_two_streams(lm, gpu, dtype, kind):
    """Two graphs on two streams, replayed side by side with other lengths than they were recorded with: equal bits to
    calls of their own."""
    cache, _, _ = filled(lm, 64, 16, 2, 64, kind)
    calls = []
    for i in range(2):
        q = normal(3, 8, 64, dtype=dtype, seed=i).cuda()
        table = tables([900, 900, 900], 16, 64, seed=i).cuda()
        calls.append((q, table, torch.tensor([900, 1, 30], dtype=torch.int32).cuda()))
    news = [torch.tensor(x, dtype=torch.int32).cuda() for x in ([1, 900, 500], [0, 64, 899])]
    want = [[lm.decode_attention(q, cache, t, n) for n in news] for q, t, _ in calls]
    torch.cuda.synchronize()
    streams, graphs, got = [torch.cuda.Stream() for _ in calls], [], []
    try:
        for s, (q, t, n) in zip(streams, calls):
            gpu.set_stream(s)
            with torch.cuda.stream(s):
                lm.decode_attention(q, cache, t, n)
                s.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=s):
                    got.append(lm.decode_attention(q, cache, t, n))
                graphs.append(graph)
        for i, new in enumerate(news):
            for (_, _, n), o in zip(calls, got):
                n.copy_(new)
                o.fill_(7)
            torch.cuda.synchronize()
            for _ in range(5):
                for s, graph in zip(streams, graphs):
                    with torch.cuda.stream(s):
                        graph.replay()
            torch.cuda.synchronize()
            for o, w in zip(got, want):
                assert torch.equal(o, w[i])
    finally:
        gpu.set_stream(torch.cuda.current_stream())


def test_decode_recorded_by_the_library(lm, gpu):
    """Between mtxc_graph_begin and mtxc_graph_end the thread's workspace holds the partial sums."""
    import ctypes as C

    from matrix_b200 import _abi

    lib = _abi.lib()
    cache, k, v = filled(lm, 64, 16, 2, 64, torch.bfloat16)
    q, table = normal(1, 8, 64, dtype=torch.bfloat16), tables([900], 16, 64)
    args = (q.cuda(), cache, table.cuda(), torch.tensor([900], dtype=torch.int32).cuda())
    out = torch.zeros_like(args[0])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        gpu.set_stream(side)
        with torch.cuda.stream(side):
            recording, graph = C.c_int(7), C.c_void_p()
            _abi.check(lib.mtxc_graph_begin())
            _abi.check(lib.mtxc_graph_recording(C.byref(recording)))
            lm.decode_attention(*args, out=out)
            _abi.check(lib.mtxc_graph_end(C.byref(graph)))
            assert recording.value == 1
            _abi.check(lib.mtxc_graph_recording(C.byref(recording)))
            assert recording.value == 0
            _abi.check(lib.mtxc_graph_launch(graph))
            side.synchronize()
            _abi.check(lib.mtxc_graph_destroy(graph))
    finally:
        gpu.set_stream(torch.cuda.current_stream())
    att.assert_close(out, *att.decode(q.double(), k, v, table, [900], 0.125, torch.bfloat16))


def test_decode_workspace_refusal(lm, gpu):
    """Partial sums that do not fit the thread's workspace: refused, and nothing is written."""
    import ctypes as C

    from matrix_b200 import _abi

    lib = _abi.lib()
    size = C.c_size_t()
    q = torch.ones(1, 2, 64, device="cuda")
    out, n = torch.full_like(q, 7.0), torch.ones(1, dtype=torch.int32, device="cuda")
    cache, table = lm.kv_cache(1, 16, 1, 64, torch.float32), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    strides = [s for t in cache[:2] for s in t.stride()[:3]]
    args = _abi.DECODE_ATTENTION_ARGS.pack(1, 16, 1, 64, 0, cache.keys.data_ptr(), cache.values.data_ptr(), *strides, 0, 0,
                                           *[0] * 6, 1, 1, 2, 0.125, q.data_ptr(), *q.stride()[:2], out.data_ptr(),
                                           *out.stride()[:2], table.data_ptr(), 1, n.data_ptr(), 0, 0)
    _abi.check(lib.mtxc_decode_attention_workspace(0, args, C.byref(size)))
    old = C.c_size_t()
    _abi.check(lib.mtxc_workspace_size(C.byref(old)))
    small = torch.empty(256, dtype=torch.uint8, device="cuda")
    large = torch.empty(old.value, dtype=torch.uint8, device="cuda")
    assert size.value > 256
    try:
        _abi.check(lib.mtxc_set_workspace(small.data_ptr(), 256))
        assert lib.mtxc_decode_attention(0, args) == _abi.ERR_WORKSPACE
        torch.cuda.synchronize()
        assert (out == 7).all()
    finally:
        KEPT.append(large)  # the thread's workspace from here on
        _abi.check(lib.mtxc_set_workspace(large.data_ptr(), large.numel()))
    _abi.check(lib.mtxc_decode_attention(0, args))
    _abi.check(lib.mtxc_sync())
    assert (out == 0).all()


@pytest.mark.parametrize("shape", [(0, 4), (3, 0)])
def test_decode_empty(lm, shape):
    cache = lm.kv_cache(2, 4, 2, 64, torch.bfloat16)
    q = torch.empty(*shape, 64, dtype=torch.bfloat16, device="cuda")
    got = lm.decode_attention(q, cache, torch.zeros(shape[0], 1, dtype=torch.int32, device="cuda"),
                              torch.ones(shape[0], dtype=torch.int32, device="cuda"))
    assert got.shape == q.shape
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    got = lm.decode_attention(q, cache, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda"))
    assert not got.any()
    got = lm.decode_attention(q, lm.kv_cache(0, 4, 2, 64, torch.bfloat16), torch.zeros(2, 1, dtype=torch.int32, device="cuda"),
                              torch.ones(2, dtype=torch.int32, device="cuda"))
    assert not got.any()


# ------------------------------------------------------------------------------------------
# Prompts
# ------------------------------------------------------------------------------------------
def starts_of(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def check_prompt(lm, dtype, lengths, qh, kh, head, k_lengths=None, causal=True, scale=None, seed=0, std=1.0, tail=0):
    starts = starts_of(lengths)
    k_starts = starts if k_lengths is None else starts_of(k_lengths)
    q = normal(starts[-1] + tail, qh, head, dtype=dtype, seed=seed, std=std)
    k = normal(k_starts[-1] + tail, kh, head, dtype=dtype, seed=seed + 1, std=std)
    v = normal(k_starts[-1] + tail, kh, head, dtype=dtype, seed=seed + 2)
    dev = [torch.tensor(s, dtype=torch.int32).cuda() for s in (starts, k_starts)]
    got = lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), dev[0], k_starts=None if k_lengths is None else dev[1],
                              scale=scale, causal=causal)
    s = head ** -0.5 if scale is None else scale
    want, bound = att.prompt(q.double(), k.double(), v.double(), starts, k_starts, s, causal, dtype)
    n = starts[-1]
    att.assert_close(got[:n], want[:n], bound[:n], f"{dtype} {lengths} {k_lengths} {qh}/{kh} x {head} causal {causal}")
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head", [1, 3, 8, 16, 40, 64, 66, 72, 80, 96, 112, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_heads(lm, dtype, head, causal):
    check_prompt(lm, dtype, [1, 130, 0, 65, 17], 4, 2, head, causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[1], [2], [63], [64], [65], [127], [128], [129], [255], [256], [257], [383, 385], [513],
                                     [1] * 70, [0, 0], [0, 5, 0], list(range(0, 140, 9)), [700]])
@pytest.mark.parametrize("head", [64, 128])
def test_prompt_lengths(lm, dtype, lengths, head):
    check_prompt(lm, dtype, lengths, 3, 1, head)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("qh,kh", [(1, 1), (5, 5), (7, 1), (16, 2), (40, 8)])
def test_prompt_groups(lm, dtype, qh, kh):
    check_prompt(lm, dtype, [150, 70], qh, kh, 64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_prefixes(lm, dtype, head, causal):
    """More keys than queries (a prefix), fewer (rows that see nothing give 0), none."""
    lengths, k_lengths = [5, 200, 130, 40, 300, 7], [305, 201, 130, 0, 100, 128]
    got = check_prompt(lm, dtype, lengths, 4, 2, head, k_lengths, causal)
    assert not got[335:375].any()  # no keys
    if causal:
        assert not got[375:575].any()  # the first 200 of 300 queries over 100 keys


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head", [64, 128, 256])
def test_prompt_long(lm, dtype, head):
    """Many tiles of keys, on both sides of the diagonal, with peaked scores."""
    check_prompt(lm, dtype, [1500, 1100], 2, 1, head, [1900, 1100])
    check_prompt(lm, dtype, [900], 2, 1, head, scale=1.5, std=2.0)
    check_prompt(lm, dtype, [900], 2, 1, head, scale=-0.5)
    check_prompt(lm, dtype, [300], 2, 1, head, scale=0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head", [64, 128, 256])
def test_prompt_a_growing_maximum(lm, dtype, head):
    """Scores that rise along the keys by far more than any bound on what is kept between maxima: every tile rescales."""
    n = 700
    q = torch.ones(n, 1, head).to(dtype)
    k = (torch.arange(n)[:, None, None] / n * torch.ones(1, 1, head)).to(dtype)
    v = normal(n, 1, head, dtype=dtype)
    starts = torch.tensor([0, n], dtype=torch.int32)
    for scale in (1.0, -1.0, 8.0):
        got = lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts.cuda(), scale=scale)
        want, bound = att.prompt(q.double(), k.double(), v.double(), [0, n], [0, n], scale, True, dtype)
        att.assert_close(got, want, bound, f"{dtype} {scale}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head", [64, 128, 100, 256])
def test_prompt_what_is_not_seen_does_not_count(lm, dtype, head):
    """NaN and infinities in later tokens, in other sequences and behind the last one."""
    lengths = [200, 150, 64]
    starts = starts_of(lengths)
    n = starts[-1]
    q, k, v = (normal(n + 100, 2, head, dtype=dtype, seed=i) for i in range(3))
    clean = [x.clone() for x in (q, k, v)]
    bad = [180, 199, 300, 414, 415, 500]
    for i, b in enumerate(bad):
        k[b, :, i % head] = float("nan") if i % 2 else float("inf")
        v[b, :, :] = float("inf") if i % 2 else float("nan")
    v[199, :, 1] = -float("inf")
    q[n:] = float("nan")
    dev = torch.tensor(starts, dtype=torch.int32).cuda()
    for causal in (True, False):
        got = lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), dev, causal=causal)
        want, bound = att.prompt(*(x.double() for x in clean), starts, starts, head ** -0.5, causal, dtype)
        # rows that see none of them
        rows = torch.ones(n, dtype=torch.bool)
        for b in bad:
            for a, e in zip(starts, starts[1:]):
                if a <= b < e:
                    rows[(b if causal else a):e] = False
        assert rows.sum() == (180 + 100 + 64 if causal else 64)
        att.assert_close(got[:n][rows], want[:n][rows], bound[:n][rows], f"{causal}")
        assert torch.isnan(got[:n][~rows].float()).any(-1).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("head", [64, 128, 256])
def test_prompt_infinite_values_that_are_seen(lm, dtype, head):
    """An infinity among the values reaches the elements of the rows that see it, and no others."""
    n = 300
    q, k, v = (normal(n, 1, head, dtype=dtype, seed=i) for i in range(3))
    clean = v.clone()
    v[270, 0, 3], v[280, 0, 3], v[20, 0, 5], v[290, 0, 7] = float("inf"), -float("inf"), float("inf"), float("nan")
    got = lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), torch.tensor([0, n], dtype=torch.int32).cuda())
    want, bound = att.prompt(q.double(), k.double(), clean.double(), [0, n], [0, n], head ** -0.5, True, dtype)
    want[270:280, 0, 3], want[280:, 0, 3], want[20:, 0, 5], want[290:, 0, 7] = torch.inf, torch.nan, torch.inf, torch.nan
    att.assert_close(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_infinite_scores(lm, dtype):
    """Keys of score -infinity get no weight; rows that see nothing else, and rows with a NaN, are NaN."""
    n, head = 200, 64
    q, k, v = (normal(n, 1, head, dtype=dtype, seed=i) for i in range(3))
    q = q.abs() + 0.125
    clean = k.clone()
    k[:3, 0, 5] = -float("inf")
    k[190, 0, 9] = float("nan")
    got = lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), torch.tensor([0, n], dtype=torch.int32).cuda())
    seen = (torch.arange(n) <= torch.arange(n)[:, None]) & (torch.arange(n) >= 3)
    want, bound = att.attend(q[:, 0].double(), clean[:, 0].double(), v[:, 0].double(), head ** -0.5, seen, dtype)
    want[:3], want[190:] = torch.nan, torch.nan
    att.assert_close(got[:, 0], want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head", [64, 128, 60])
def test_prompt_layouts(lm, dtype, head):
    """Slices of one tensor of queries, keys and values, heads before tokens, misaligned, rows behind the last sequence
    left as they were, the output over the queries."""
    lengths = [140, 60]
    starts = starts_of(lengths)
    dev = torch.tensor(starts, dtype=torch.int32).cuda()
    for pad, lo in ((0, 0), (8, 8), (3, 1)):
        base = normal(230, 8, head + pad, dtype=dtype).cuda()
        qkv = base[..., lo:lo + head]
        q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
        want, bound = att.prompt(*(t.cpu().double() for t in (q, k, v)), starts, starts, head ** -0.5, True, dtype)
        att.assert_close(lm.prompt_attention(q, k, v, dev)[:200], want[:200], bound[:200], f"{pad} {lo}")
        t = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
        att.assert_close(lm.prompt_attention(*t, dev)[:200], want[:200], bound[:200], f"{pad} {lo}")
        before = base.clone()
        assert lm.prompt_attention(q, k, v, dev, out=q) is q
        att.assert_close(q[:200], want[:200], bound[:200], f"{pad} {lo}")
        before[:200, :4, lo:lo + head] = q[:200]
        assert torch.equal(before, base)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_starts_outside(lm, dtype):
    """starts and k_starts are cut to the tokens that there are; a sequence that ends before it begins is empty."""
    q, k, v = (normal(100, 2, 64, dtype=dtype, seed=i) for i in range(3))
    out = torch.full((100, 2, 64), 7.0, dtype=dtype, device="cuda")
    starts = torch.tensor([-5, 40, 40, 1 << 30], dtype=torch.int32).cuda()
    lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), starts, out=out)
    want, bound = att.prompt(q.double(), k.double(), v.double(), [0, 40, 40, 100], [0, 40, 40, 100], 0.125, True, dtype)
    att.assert_close(out, want, bound)
    out.fill_(7.0)
    lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), torch.tensor([60, 20], dtype=torch.int32).cuda(), out=out)
    assert (out == 7).all()
    lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), torch.tensor([10], dtype=torch.int32).cuda(), out=out)
    assert (out == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_empty(lm, dtype):
    starts = torch.tensor([0, 0], dtype=torch.int32).cuda()
    q = torch.empty(0, 2, 64, dtype=dtype, device="cuda")
    assert lm.prompt_attention(q, q, q, starts).shape == q.shape
    q = torch.ones(3, 2, 64, dtype=dtype, device="cuda")
    none = torch.empty(0, 1, 64, dtype=dtype, device="cuda")
    got = lm.prompt_attention(q, none, none, torch.tensor([0, 3], dtype=torch.int32).cuda(), k_starts=starts)
    assert not got.any()
    empty = torch.empty(3, 0, 64, dtype=dtype, device="cuda")
    assert lm.prompt_attention(empty, q, q, torch.tensor([0, 3], dtype=torch.int32).cuda()).shape == empty.shape


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_recorded_and_repeated(lm, gpu, dtype):
    """Equal calls give equal bits; a graph recorded on a stream of the caller's takes other lengths and inputs."""
    q, k, v = (normal(300, 4, 128, dtype=dtype, seed=i).cuda() for i in range(3))
    starts = torch.tensor([0, 300, 300], dtype=torch.int32).cuda()
    other = torch.tensor([0, 111, 300], dtype=torch.int32).cuda()
    want = lm.prompt_attention(q, k, v, other)
    for _ in range(3):
        assert torch.equal(lm.prompt_attention(q, k, v, other), want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    try:
        gpu.set_stream(side)
        with torch.cuda.stream(side):
            lm.prompt_attention(q, k, v, starts)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                got = lm.prompt_attention(q, k, v, starts)
            starts.copy_(other)
            graph.replay()
            side.synchronize()
            assert torch.equal(got, want)
    finally:
        gpu.set_stream(torch.cuda.current_stream())


def test_prompt_and_decode_agree(lm):
    """The last row of a prompt and a token over the same keys and values in a cache."""
    n, page = 333, 16
    for dtype in TYPES:
        q, k, v = normal(n, 8, 64, dtype=dtype), normal(n, 2, 64, dtype=dtype, seed=1), normal(n, 2, 64, dtype=dtype, seed=2)
        cache = lm.kv_cache(30, page, 2, 64, dtype)
        table = torch.randperm(30, generator=torch.Generator().manual_seed(0))[:21].to(torch.int32)
        at = torch.arange(n)
        slots = table[at // page] * page + at % page
        lm.cache_write(cache, k.cuda(), v.cuda(), slots.cuda())
        a = lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), torch.tensor([0, n], dtype=torch.int32).cuda())[-1]
        b = lm.decode_attention(q[-1:].cuda(), cache, table[None].cuda(), torch.tensor([n], dtype=torch.int32).cuda())[0]
        want, bound = att.prompt(q.double(), k.double(), v.double(), [0, n], [0, n], 0.125, True, dtype)
        att.assert_close(a, want[-1], bound[-1])
        att.assert_close(b, want[-1], bound[-1])


def test_threads(lm, gpu):
    """Threads with streams of their own, calls of different shared memory and workspaces."""
    from matrix_b200 import backend

    works = []
    for dtype, kind, head in ((torch.float32, torch.float32, 64), (torch.float32, torch.float32, 256), (torch.bfloat16, torch.bfloat16, 128),
                              (torch.bfloat16, E4M3, 128)):
        cache, _, _ = filled(lm, 32, 16, 2, head, kind)
        q = normal(2, 8, head, dtype=dtype).cuda()
        table, n = tables([500, 300], 16, 32).cuda(), torch.tensor([500, 300], dtype=torch.int32).cuda()
        p = [normal(200, h, head, dtype=dtype, seed=h).cuda() for h in (4, 2, 2)]
        starts = torch.tensor([0, 150, 200], dtype=torch.int32).cuda()
        works.append(lambda q=q, cache=cache, table=table, n=n, p=p, starts=starts:
                     (lm.decode_attention(q, cache, table, n), lm.prompt_attention(*p, starts)))
    want = [w() for w in works]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            torch.cuda.set_device(0)
            backend.init(0)
            s = torch.cuda.Stream()
            backend.set_stream(s)
            with torch.cuda.stream(s):
                for _ in range(30):
                    got = works[i]()
                    s.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(works))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("qh,kh", [(4, 2), (3, 1), (6, 2)])
def test_prompt_an_infinite_value_for_some_heads(lm, dtype, qh, kh):
    """Non-finite values of one key head, seen by the second of the heads that share it too, beside another key head's finite
    ones."""
    n, head = 200, 64
    q, k, v = normal(n, qh, head, dtype=dtype), normal(n, kh, head, dtype=dtype, seed=1), normal(n, kh, head, dtype=dtype, seed=2)
    clean = v.clone()
    v[150, 0, 3], v[199, 0, 9] = float("inf"), float("nan")
    got = lm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), torch.tensor([0, n], dtype=torch.int32).cuda())
    want, bound = att.prompt(q.double(), k.double(), clean.double(), [0, n], [0, n], head ** -0.5, True, dtype)
    group = qh // kh
    want[150:, :group, 3], want[199:, :group, 9] = torch.inf, torch.nan
    att.assert_close(got, want, bound)


@pytest.mark.parametrize("dtype,kind", KINDS)
def test_decode_many_rows_of_long_sequences(lm, dtype, kind):
    """More rows than a join by rows takes, and sequences long enough to be shared: joined by units, several rows each."""
    check_decode(lm, dtype, kind, [700] * 20 + [0, 3, 2000], 40, 2, 64, 16, pages=64)
    check_decode(lm, dtype, kind, [900] * 25, 28, 4, 128, 24, pages=40)
