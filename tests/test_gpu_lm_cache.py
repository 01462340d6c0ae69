"""The paged cache (mtxc_cache_write, mtxc_cache_read): what is read back has to be equal, element by element, to what was
written, or in 8 bits to its rounding to e4m3 times the least power of two that fits -- neither the scaling nor its
inverse rounds, so there is no bound but equality (a read to float16 rounds once more, to equal bits)."""
import pytest
import torch

from tests import attention_reference as att

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
E4M3 = torch.float8_e4m3fn


@pytest.fixture
def lm(gpu):
    from matrix_b200 import lm

    return lm


def normal(*shape, dtype=torch.float32, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed * 31 + sum(shape))) * std).to(dtype)


def same(a, b):
    a, b = a.cpu(), b.cpu()
    return a.shape == b.shape and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def distinct_slots(tokens, total, seed=0):
    return torch.randperm(total, generator=torch.Generator().manual_seed(seed))[:tokens]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("small", [False, True])
@pytest.mark.parametrize("head", [1, 3, 8, 64, 66, 80, 96, 128, 200, 256, 512, 1000])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 1), (5, 3, 16), (70, 2, 24), (1000, 1, 64)])
def test_write_and_read(lm, dtype, small, head, tokens, heads, page):
    pages = (tokens + page - 1) // page + 2
    cache = lm.kv_cache(pages, page, heads, head, E4M3 if small else dtype)
    k, v = normal(tokens, heads, head, dtype=dtype, std=3.0), normal(tokens, heads, head, dtype=dtype, seed=1, std=0.01)
    slots = distinct_slots(tokens, pages * page)
    lm.cache_write(cache, k.cuda(), v.cuda(), slots.to(torch.int32).cuda())
    got = lm.cache_read(cache, slots.cuda(), dtype=dtype)
    for x, y, data, exponents in ((k, got[0], cache.keys, cache.key_exponents), (v, got[1], cache.values, cache.value_exponents)):
        if not small:
            assert same(y, x)
            assert same(data.cpu()[slots // page, slots % page], x)
            continue
        want, e = att.quantise(x.double())
        assert torch.equal(exponents.cpu()[slots // page, slots % page].long(), e.long())
        assert same(y, want.to(dtype))
    # the slots that were not named keep their zeros
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots] = False
    rest = rest.nonzero()[:, 0]
    k, v = lm.cache_read(cache, rest.cuda(), dtype=dtype)
    assert not k.any() and not v.any()


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("source", TYPES)
def test_types_of_a_cache_in_8_bits(lm, source, out):
    cache = lm.kv_cache(4, 16, 2, 64, E4M3)
    k, v = normal(40, 2, 64, dtype=source, std=50.0), normal(40, 2, 64, dtype=source, seed=1, std=1e-3)
    slots = distinct_slots(40, 64).cuda()
    lm.cache_write(cache, k.cuda(), v.cuda(), slots)
    got = lm.cache_read(cache, slots, dtype=out)
    for x, y in zip((k, v), got):
        assert y.dtype == out and same(y, att.quantise(x.double())[0].to(out))
    if out == torch.bfloat16:
        assert same(lm.cache_read(cache, slots)[0], got[0])


def test_rounding_of_8_bits(lm):
    """Every row holds 448 * 2^e, so that its scale is 2^e exactly, and the borders between the type's values, a step of
    float32 to either side of them, its largest, its smallest, and what lies below."""
    values = torch.arange(127, dtype=torch.uint8).view(E4M3).double()  # 0 .. 448
    middle = (values[1:] + values[:-1]) / 2
    points = torch.cat([values, middle, torch.nextafter(middle.float(), torch.tensor(1e9)).double(),
                        torch.nextafter(middle.float(), torch.tensor(0.0)).double()])
    points = torch.cat([points, -points])
    cache = lm.kv_cache(1, 8, 1, len(points), E4M3)
    for e in (0, 1, -9, 30, -40, 96, -96):
        x = (points * 2.0 ** e).float()[None, None]
        lm.cache_write(cache, x.cuda(), x.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"))
        k, _ = lm.cache_read(cache, torch.zeros(1, dtype=torch.int32, device="cuda"), dtype=torch.float32)
        want, got_e = att.quantise(x.double())
        assert got_e.item() == e and cache.key_exponents.cpu()[0, 0, 0].item() == e
        assert same(k, want.float())


def test_scales(lm):
    """The least power of two: rows whose largest is 448 * 2^e, a step above, zero, tiny and huge; infinities and NaN,
    which do not count for it and come back as NaN."""
    tops = [448.0, 449.0, 447.0, 896.0, 0.0, 1e-30, 2.0 ** -149, 3e38, 1.0, 1.75, 1.7500001, 2.0 ** -88 * 448, 2.0 ** -87 * 448]
    x = torch.zeros(len(tops), 1, 16)
    x[:, 0, 3] = torch.tensor(tops)
    x[:, 0, 4] = -torch.tensor(tops) / 3
    cache = lm.kv_cache(2, 16, 1, 16, E4M3)
    slots = torch.arange(len(tops)).cuda()
    lm.cache_write(cache, x.cuda(), -x.cuda(), slots)
    want, e = att.quantise(x.double())
    k, v = lm.cache_read(cache, slots, dtype=torch.float32)
    assert torch.equal(cache.key_exponents.cpu().flatten(0, 1)[:len(tops)].long(), e.long())
    assert same(k, want.float()) and same(v, -want.float())
    x[2, 0, 5], x[3, 0, 6], x[4, 0, 7] = float("inf"), float("nan"), -float("inf")
    lm.cache_write(cache, x.cuda(), x.cuda(), slots)
    want, _ = att.quantise(x.double())
    assert torch.isnan(want).sum() == 3 and same(lm.cache_read(cache, slots, dtype=torch.float32)[0], want.float())


@pytest.mark.parametrize("small", [False, True])
@pytest.mark.parametrize("head", [64, 20])
def test_slots_outside_and_twice(lm, small, head):
    """Slots outside the cache are passed over and read as zeros; of several tokens of one slot the last counts, across
    the tiles of a block and the launches of a call too."""
    for tokens, total in ((7, 3), (300, 40), (20000, 700), (40000, 33)):
        pages = (total + 15) // 16
        cache = lm.kv_cache(pages, 16, 1, head, E4M3 if small else torch.float32)
        g = torch.Generator().manual_seed(tokens)
        slots = torch.randint(-3, pages * 16 + 5, (tokens,), generator=g)
        slots[1] = 1 << 40
        k = normal(tokens, 1, head)
        lm.cache_write(cache, k.cuda(), -k.cuda(), slots.cuda())
        want = torch.zeros(pages * 16, 1, head)
        inside = (slots >= 0) & (slots < pages * 16)
        for t in inside.nonzero()[:, 0].tolist():
            want[slots[t]] = k[t]
        if small:
            want = att.quantise(want.double())[0].float()
        got = lm.cache_read(cache, torch.arange(pages * 16).cuda(), dtype=torch.float32)
        assert same(got[0], want) and same(got[1], -want), (tokens, total)
    back = lm.cache_read(cache, torch.tensor([-1, 0, 1 << 35, pages * 16]).cuda(), dtype=torch.float32)
    assert same(back[0][1], want[0]) and not back[0][[0, 2, 3]].any()


@pytest.mark.parametrize("small", [False, True])
@pytest.mark.parametrize("head", [64, 72, 33])
def test_layouts(lm, small, head):
    """A cache with slots before heads, one that is a part of a larger tensor; rows that are slices, misaligned, with
    strided slots; outputs that are given."""
    dtype = torch.bfloat16
    kind = E4M3 if small else dtype
    big = torch.zeros(2, 6, 16, 5, head + 1, dtype=torch.int8 if small else dtype, device="cuda")
    big = big.view(kind)
    exponents = torch.zeros(2, 6, 16, 5, dtype=torch.int8, device="cuda") if small else [None, None]
    for lo in (0, 1):
        data = big[..., lo:lo + head]
        cache = lm.KVCache(data[0][:, :, 1:4], data[1][:, :, 1:4], *(e[:, :, 1:4] if small else None for e in exponents))
        qkv = normal(30, 9, head, dtype=dtype).cuda()
        slots = torch.stack([distinct_slots(30, 96), torch.arange(30)], 1).to(torch.int32).cuda()[:, 0]
        before = big.view(torch.int8).clone()
        lm.cache_write(cache, qkv[:, 3:6], qkv[:, 6:9], slots)
        out = torch.full((30, 8, head), 7.0, dtype=dtype, device="cuda")
        got = lm.cache_read(cache, slots, out=(out[:, 1:4], out[:, 5:8]))
        assert got[0].data_ptr() == out[:, 1:4].data_ptr()
        for i, x in ((0, qkv[:, 3:6]), (1, qkv[:, 6:9])):
            want = att.quantise(x.cpu().double())[0].to(dtype) if small else x
            assert same(got[i], want)
        assert (out[:, [0, 4]] == 7).all()
        after = big.view(torch.int8)
        changed = (after != before).view(2, 6, 16, 5, head + 1, -1).any(-1)
        assert not changed[:, :, :, [0, 4]].any() and not changed[..., head if lo == 0 else 0].any()
        big.view(torch.int8).zero_()


def test_a_cache_past_32_bits(lm):
    """Offsets of bytes and elements beyond 2^32 (a cache of 5 GB of keys and values that share no memory)."""
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("not enough memory")
    pages, page, heads, head = 40, 1024, 8, 8192 * 2 // 16
    stride = (1 << 32) // 32 + 4096
    base = torch.empty(pages * stride, dtype=torch.int8, device="cuda")
    data = torch.as_strided(base, (pages, page, heads, head), (stride, heads * head, head, 1)).view(E4M3)
    values = torch.zeros(pages, page, heads, head, dtype=torch.int8, device="cuda").view(E4M3)
    exponents = [torch.zeros(pages, page, heads, dtype=torch.int8, device="cuda") for _ in range(2)]
    cache = lm.KVCache(data, values, *exponents)
    assert (pages - 1) * stride > 1 << 32
    k = normal(20, heads, head).cuda()
    slots = distinct_slots(20, 1024).cuda() + (pages - 1) * page
    lm.cache_write(cache, k, k, slots)
    got = lm.cache_read(cache, slots, dtype=torch.float32)
    want = att.quantise(k.cpu().double())[0].float()
    assert same(got[0], want) and same(got[1], want)


@pytest.mark.parametrize("small", [False, True])
def test_empty(lm, small):
    kind = E4M3 if small else torch.float32
    cache = lm.kv_cache(2, 4, 3, 8, kind)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    lm.cache_write(cache, torch.empty(0, 3, 8, device="cuda"), torch.empty(0, 3, 8, device="cuda"), none)
    assert lm.cache_read(cache, none, dtype=torch.float32)[0].shape == (0, 3, 8)
    nothing = lm.kv_cache(0, 4, 3, 8, kind)
    slots = torch.zeros(2, dtype=torch.int32, device="cuda")
    lm.cache_write(nothing, torch.ones(2, 3, 8, device="cuda"), torch.ones(2, 3, 8, device="cuda"), slots)
    assert not lm.cache_read(nothing, slots, dtype=torch.float32)[0].any()


def test_a_recorded_write(lm, gpu):
    """A graph that stores a step's keys, replayed with other slots and keys; the cache counts as changed in place."""
    cache = lm.kv_cache(4, 16, 2, 64, E4M3)
    k, slots = normal(3, 2, 64).cuda(), torch.tensor([1, 2, 3], dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    try:
        gpu.set_stream(side)
        with torch.cuda.stream(side):
            version = cache.keys._version
            lm.cache_write(cache, k, k, slots)
            assert cache.keys._version > version and cache.value_exponents._version > 0
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                lm.cache_write(cache, k, k, slots)
                got = lm.cache_read(cache, slots, dtype=torch.float32)
            for i in range(3):
                k.copy_(normal(3, 2, 64, seed=i))
                slots.copy_(distinct_slots(3, 64, seed=i))
                graph.replay()
                side.synchronize()
                assert same(got[0], att.quantise(normal(3, 2, 64, seed=i).double())[0].float())
    finally:
        gpu.set_stream(torch.cuda.current_stream())
