"""Rotary positions (mtxc_rotary) against the rotation in 64 bits.

The bound: the angle's fraction of a turn, at most half, is rounded once to 24 bits (2 pi 2^-25 radians), sine and
cosine are within 2 ulp, and two products and a sum follow: less than 2^-20 of |x| + |y|.  The angle itself, up to four roundings
in 64 bits between the kernel and the formula, differs by at most 2^-51 of it."""
import pytest
import torch

from tests import lm_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
WORK = 2.0 ** -20


@pytest.fixture
def lm(gpu):
    from matrix_b200 import lm

    return lm


def normal(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(dtype)


def check(lm, q, k, positions, freq, what="", scale=1.0, interleaved=False, inverse=False, **more):
    """q, k: device tensors [batch, length, heads, head] (k may be None); positions [batch, length] on the host."""
    got = lm.rotary(q, k, positions.cuda(), freq.cuda(), scale=scale, interleaved=interleaved, inverse=inverse, **more)
    for x, y in ((q, got[0]), (k, got[1])):
        if x is None:
            assert y is None
            continue
        want, mag = ref.rotary(x.cpu().double(), positions, freq, torch.tensor(scale).double().item(), interleaved, inverse)
        angle = positions.double().abs().max().item() * (freq.max().item() if len(freq) else 0.0)
        ref.assert_within(y, want, mag, f"{what} {tuple(x.shape)} {x.dtype}", WORK + 2.0 ** -51 * angle)
        r = 2 * len(freq)
        assert torch.equal(y[..., r:], x[..., r:])
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head,part", [(2, 2), (3, 2), (8, 8), (16, 6), (64, 64), (65, 64), (80, 32), (96, 96), (100, 50), (128, 128),
                                       (128, 64), (192, 64), (256, 256), (512, 512), (1024, 1024), (64, 0)])
def test_heads_and_parts(lm, dtype, interleaved, head, part):
    freq = lm.rotary_frequencies(part, device="cpu")[0]
    for batch, length, qh, kh in ((1, 1, 1, 1), (2, 5, 6, 2), (3, 17, 7, 1), (2, 9, 4, 0)):
        q = normal(batch, length, qh, head, dtype=dtype).cuda()
        k = normal(batch, length, kh, head, dtype=dtype).cuda() if kh else None
        positions = torch.randint(0, 4096, (batch, length), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
        check(lm, q, k, positions, freq, f"part {part}", interleaved=interleaved)
        check(lm, q, k, positions, freq, f"part {part}", scale=1.25, interleaved=interleaved, inverse=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("top", [1, 1 << 17, 10 ** 6, 2 ** 31 - 1])
def test_long_positions(lm, dtype, interleaved, top):
    freq, scale = lm.rotary_frequencies(128, 500000.0, scaling="by_parts", factor=32, original_length=8192, device="cpu")
    positions = top - torch.arange(40, dtype=torch.int64).view(1, 40).clamp(max=top)
    q = normal(1, 40, 3, 128, dtype=dtype).cuda()
    check(lm, q, None, positions, freq, f"top {top}", scale=scale, interleaved=interleaved)
    check(lm, q, None, positions.to(torch.int32), freq, f"top {top}", scale=scale, interleaved=interleaved)
    check(lm, q, None, -positions, freq, f"top -{top}", scale=scale, interleaved=interleaved)


def test_positions_past_32_bits(lm):
    freq = lm.rotary_frequencies(64, device="cpu")[0]
    check(lm, normal(1, 3, 2, 64).cuda(), None, torch.tensor([[1 << 33, (1 << 40) + 1, 5]]), freq)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts(lm, dtype, interleaved):
    """Heads before tokens, slices of one tensor of queries, keys and values, misaligned bases, expanded keys."""
    freq = lm.rotary_frequencies(64, device="cpu")[0]
    positions = torch.arange(12, dtype=torch.int32).view(1, 12).expand(2, 12) + 100
    q = normal(2, 6, 12, 64, dtype=dtype).cuda().transpose(1, 2)
    k = normal(2, 2, 12, 64, dtype=dtype).cuda().transpose(1, 2)
    got = check(lm, q, k, positions, freq, interleaved=interleaved)
    assert got[0].stride() == q.stride()
    for head in (64, 70, 65):
        qkv = normal(2, 12, 10, head, dtype=dtype).cuda()
        check(lm, qkv[:, :, :6], qkv[:, :, 6:8], positions, freq, interleaved=interleaved)
    for start in (1, 3, 4, 8):
        base = normal(start + 2 * 12 * 6 * 72, dtype=dtype).cuda()
        q = torch.as_strided(base, (2, 12, 6, 64), (12 * 6 * 72, 6 * 72, 72, 1), start)
        check(lm, q, None, positions, freq, interleaved=interleaved)
    one = normal(2, 12, 1, 64, dtype=dtype).cuda().expand(2, 12, 4, 64)
    check(lm, one, one[:, :, :2], positions, freq, interleaved=interleaved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("part", [64, 32])
def test_in_place_and_into_strided_outputs(lm, dtype, interleaved, part):
    freq = lm.rotary_frequencies(part, device="cpu")[0]
    positions = torch.arange(7, dtype=torch.int32).view(1, 7)
    qkv = normal(1, 7, 9, 64, dtype=dtype).cuda()
    want = qkv.clone()
    q, k = lm.rotary(qkv[:, :, :5], qkv[:, :, 5:7], positions.cuda(), freq.cuda(), interleaved=interleaved)
    want[:, :, :5], want[:, :, 5:7] = q, k
    views = qkv[:, :, :5], qkv[:, :, 5:7]
    got = lm.rotary(*views, positions.cuda(), freq.cuda(), interleaved=interleaved, out=views)
    assert got[0] is views[0] and torch.equal(qkv, want)


def test_shapes_of_positions(lm):
    freq = lm.rotary_frequencies(32, device="cpu")[0]
    q = normal(3, 5, 2, 32).cuda()
    pos = torch.tensor([4, 9, 2, 7, 7], dtype=torch.int64)
    want = lm.rotary(q, None, pos.expand(3, 5).contiguous().cuda(), freq.cuda())[0]
    assert torch.equal(lm.rotary(q, None, pos.cuda(), freq.cuda())[0], want)
    assert torch.equal(lm.rotary(q, None, pos[None].cuda(), freq.cuda())[0], want)
    assert torch.equal(lm.rotary(q[1], None, pos.cuda(), freq.cuda())[0], want[1])
    wide = torch.stack([pos, pos + 1], 1).cuda()[:, 0]  # strided positions
    assert torch.equal(lm.rotary(q, None, wide, freq.cuda())[0], want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_undoes_and_is_the_gradient(lm, interleaved):
    """<rotate(x), g> = <x, inverse(g)>: the backward pass, scale included; and against differences of the
    formula in 64 bits, which is linear, so that one difference of any step is exact."""
    freq, scale = lm.rotary_frequencies(48, scaling="by_parts", factor=4, original_length=100, device="cpu")
    positions = torch.randint(0, 1000, (2, 3), generator=torch.Generator().manual_seed(0), dtype=torch.int32)
    x, g = normal(2, 3, 2, 50), normal(2, 3, 2, 50, seed=9)
    how = dict(scale=scale, interleaved=interleaved)
    back = lm.rotary(g.cuda(), None, positions.cuda(), freq.cuda(), inverse=True, **how)[0].cpu().double()
    s = torch.tensor(scale).double().item()
    f = lambda v: (ref.rotary(v, positions, freq, s, interleaved, False)[0] * g.double()).sum()  # noqa: E731
    base = f(x.double())
    for i in range(0, x.numel(), 7):
        v = x.double().clone()
        v.view(-1)[i] += 1.0
        want = (f(v) - base).item()
        assert abs(back.view(-1)[i].item() - want) <= WORK * 8 * s
    turned = lm.rotary(x.cuda(), None, positions.cuda(), freq.cuda(), interleaved=interleaved)[0]
    again = lm.rotary(turned, None, positions.cuda(), freq.cuda(), interleaved=interleaved, inverse=True)[0]
    assert (again.cpu() - x).abs().max() <= 2 * WORK * 8


def test_special_values_stay_in_their_pair(lm):
    freq = lm.rotary_frequencies(64, device="cpu")[0]
    x = normal(1, 4, 2, 64)
    x[0, 1, 0, 5] = float("nan")
    x[0, 2, 1, 40] = float("inf")
    y = lm.rotary(x.cuda(), None, torch.arange(4, dtype=torch.int32).cuda() + 3, freq.cuda())[0].cpu()
    bad = ~torch.isfinite(y)
    assert bad.sum() == 4 and bad[0, 1, 0, 5] and bad[0, 1, 0, 37] and bad[0, 2, 1, 8] and bad[0, 2, 1, 40]


@pytest.mark.parametrize("shape", [(0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64)])
def test_empty(lm, shape):
    q, _ = lm.rotary(torch.empty(shape, device="cuda"), None, torch.zeros(shape[1], dtype=torch.int32, device="cuda"),
                     lm.rotary_frequencies(64)[0])
    assert q.shape == shape


def test_long_offsets(lm):
    """Tokens further than 2^32 bytes apart."""
    freq = lm.rotary_frequencies(64, device="cpu")[0]
    base = torch.zeros((3 << 30) + 128, dtype=torch.float16, device="cuda")
    q = torch.as_strided(base, (1, 4, 2, 64), (0, 1 << 30, 64, 1))
    q.copy_(normal(1, 4, 2, 64, dtype=torch.float16))
    k = q.contiguous()
    positions = torch.arange(4, dtype=torch.int32).view(1, 4)
    check(lm, k, None, positions, freq)
    want = lm.rotary(k, None, positions.cuda(), freq.cuda())[0]
    lm.rotary(q, None, positions.cuda(), freq.cuda(), out=(q, None))
    assert torch.equal(q, want)


def test_many_tokens(lm):
    """More tokens than blocks, queries and keys, against the same rotation token by token."""
    freq, scale = lm.rotary_frequencies(128, device="cpu")
    q, k = normal(2, 6000, 4, 128, dtype=torch.bfloat16).cuda(), normal(2, 6000, 1, 128, dtype=torch.bfloat16).cuda()
    positions = torch.arange(6000, dtype=torch.int32).expand(2, 6000) + torch.tensor([[0], [77]], dtype=torch.int32)
    check(lm, q, k, positions.contiguous(), freq)


def test_another_stream(lm, gpu):
    freq = lm.rotary_frequencies(64)[0]
    q = normal(2, 50, 4, 64).cuda()
    pos = torch.arange(50, dtype=torch.int32, device="cuda")
    want = lm.rotary(q, None, pos, freq)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    try:
        gpu.set_stream(side)
        got = lm.rotary(q, None, pos, freq)[0]
        side.synchronize()
        assert torch.equal(got, want)
    finally:
        torch.cuda.synchronize()
        gpu.set_stream(torch.cuda.current_stream())


def test_refusals(lm):
    from matrix_b200 import MtxcError, _abi

    q = torch.zeros(2, 3, 4, 64, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    freq = lm.rotary_frequencies(64)[0]
    for call in (lambda: lm.rotary(q[0, 0], None, pos, freq), lambda: lm.rotary(q, q[:, :2], pos, freq),
                 lambda: lm.rotary(q, q.half(), pos, freq), lambda: lm.rotary(q, q[..., :32], pos, freq),
                 lambda: lm.rotary(q, None, pos[:2], freq), lambda: lm.rotary(q, None, pos.float(), freq),
                 lambda: lm.rotary(q, None, pos, freq.float()), lambda: lm.rotary(q.transpose(2, 3), None, pos, freq),
                 lambda: lm.rotary(q, None, pos, freq.cpu()), lambda: lm.rotary(q, None, pos, freq, out=(q[:1], None))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(MtxcError) as e:  # more frequencies than half a head
        lm.rotary(q, None, pos, lm.rotary_frequencies(66)[0])
    assert e.value.code == _abi.ERR_INVALID_ARGUMENT
    with pytest.raises(MtxcError) as e:
        lm.rotary(q.int(), None, pos, freq)
    assert e.value.code == _abi.ERR_UNSUPPORTED_DTYPE


@pytest.mark.parametrize("interleaved", [False, True])
def test_heads_that_overlap(lm, interleaved):
    """Heads that are windows of one buffer, a stride of one element apart: the output is a tensor of its own."""
    freq = lm.rotary_frequencies(8, device="cpu")[0]
    base = normal(64).cuda()
    for shape, strides in (((1, 5, 2, 8), (64, 1, 8, 1)), ((1, 3, 4, 8), (64, 0, 1, 1)), ((2, 3, 2, 8), (1, 16, 8, 1))):
        x = torch.as_strided(base, shape, strides)
        positions = torch.arange(shape[1], dtype=torch.int32).expand(shape[:2]).contiguous()
        check(lm, x, x, positions, freq, f"strides {strides}", interleaved=interleaved)


def test_outputs_that_overlap_are_refused(lm):
    """Two elements of an output at one address."""
    freq, pos = lm.rotary_frequencies(64)[0], torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 3, 4, 64, device="cuda")
    base = torch.zeros(4096, device="cuda")
    for strides in ((0, 256, 64, 1), (768, 0, 64, 1), (768, 256, 0, 1), (768, 256, 63, 1), (768, 255, 64, 1), (767, 256, 64, 1),
                    (64, 384, 128, 1)):
        with pytest.raises(ValueError, match="overlap"):
            lm.rotary(q, None, pos, freq, out=(torch.as_strided(base, q.shape, strides), None))
    for strides in ((768, 256, 64, 1), (1024, 256, 64, 1), (64, 128, 512, 1), (64, 512, 128, 1)):  # orders of the axes, and room between
        out = torch.as_strided(torch.zeros(4096, device="cuda"), q.shape, strides)
        assert lm.rotary(q + 1, None, pos, freq, out=(out, None))[0] is out
        assert torch.equal(out, lm.rotary(q + 1, None, pos, freq)[0])


def test_one_tensor_for_queries_and_keys_is_refused(lm):
    from matrix_b200 import MtxcError, _abi

    freq, pos = lm.rotary_frequencies(64)[0], torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 3, 4, 64, device="cuda")
    out = torch.empty_like(q)
    with pytest.raises(MtxcError) as e:
        lm.rotary(q, q, pos, freq, out=(out, out))
    assert e.value.code == _abi.ERR_INVALID_ARGUMENT
