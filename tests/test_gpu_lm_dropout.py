"""Dropout (mtxc_dropout): the mask bit for bit against the generator in numpy, the values against one product
in 32 bits rounded once, at sizes, strides and alignments where indexing can go wrong."""
import numpy as np
import pytest
import torch

from tests import lm_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture
def lm(gpu):
    from matrix_b200 import lm

    return lm


def expected(x, p, seed, offset):
    """x * 65536 / kept in 32 bits where kept, else 0, rounded to x's dtype."""
    rows, width = (x.numel() // x.shape[-1], x.shape[-1]) if x.numel() else (0, 1)
    kept = round((1 - p) * 65536)
    mask = torch.from_numpy(ref.lanes(seed, offset, rows, width) < kept).view(x.shape)
    scale = torch.tensor(65536 / kept if kept else 0.0, dtype=torch.float64).float()
    return torch.where(mask, x.float() * scale, 0.0).to(x.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 7), (3, 8), (5, 9), (2, 31), (4, 64), (7, 255), (3, 257), (2, 1000),
                                        (33, 129), (1, 4099), (300, 2048), (2, 70001), (1000, 3), (1, 1 << 20)])
def test_values_and_mask(lm, dtype, rows, width):
    x = torch.randn(rows, width, generator=torch.Generator().manual_seed(rows * 7 + width)).to(dtype)
    for p, seed, offset in ((0.1, 1, 0), (0.5, 0x123456789ABCDEF0, 0xFEDCBA9876543210), (0.999, 5, 1 << 32)):
        got = lm.dropout(x.cuda(), p, seed, offset).cpu()
        assert torch.equal(got, expected(x, p, seed, offset)), (p, seed, offset)


@pytest.mark.parametrize("dtype", TYPES)
def test_ends_of_the_probability(lm, dtype):
    x = torch.randn(9, 77, generator=torch.Generator().manual_seed(0)).to(dtype)
    x[0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0])
    got = lm.dropout(x.cuda(), 0.0, 3, 4).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(x)) and torch.equal(got.nan_to_num(9.0), x.nan_to_num(9.0))
    assert torch.equal(lm.dropout(x.cuda(), 1.0, 3, 4).cpu(), torch.zeros_like(x))  # dropped NaN and inf are zeros
    assert torch.equal(lm.dropout(x[1:].cuda(), 1e-6, 3, 4).cpu(), x[1:])  # fewer than half of 2^-16: nothing dropped


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,stride,start", [(64, 72, 0), (64, 64, 1), (100, 131, 3), (33, 40, 5), (8, 9, 0), (2048, 2056, 8),
                                                (1000, 1001, 1)])
def test_strides_and_alignment(lm, dtype, width, stride, start):
    rows = 6
    base = torch.randn(start + rows * stride, generator=torch.Generator().manual_seed(width)).to(dtype)
    x = torch.as_strided(base, (rows, width), (stride, 1), start)
    dbase = base.cuda()
    view = torch.as_strided(dbase, (rows, width), (stride, 1), start)
    want = expected(x, 0.3, 11, 12)
    assert torch.equal(lm.dropout(view, 0.3, 11, 12).cpu(), want)
    # into a strided output, whose gaps stay as they are, and in place
    obase = torch.full_like(dbase, 7.0)
    out = torch.as_strided(obase, (rows, width), (stride, 1), start)
    lm.dropout(view, 0.3, 11, 12, out=out)
    check = torch.full_like(base, 7.0)
    torch.as_strided(check, (rows, width), (stride, 1), start).copy_(want)
    assert torch.equal(obase.cpu(), check)
    lm.dropout(view, 0.3, 11, 12, out=view)
    check = base.clone()
    torch.as_strided(check, (rows, width), (stride, 1), start).copy_(want)
    assert torch.equal(dbase.cpu(), check)


def test_leading_axes_fold_and_broadcast_rows(lm):
    x = torch.randn(3, 4, 5, 24, generator=torch.Generator().manual_seed(2))
    assert torch.equal(lm.dropout(x.cuda(), 0.25, 1, 2).cpu(), expected(x, 0.25, 1, 2))
    one = torch.randn(1, 24).expand(6, 24)  # one row read six times: six masks
    got = lm.dropout(one.cuda()[:1].expand(6, 24), 0.25, 1, 2).cpu()
    assert torch.equal(got, expected(one, 0.25, 1, 2))
    v = torch.randn(100)
    assert torch.equal(lm.dropout(v.cuda(), 0.25, 1, 2).cpu(), expected(v[None], 0.25, 1, 2)[0])
    s = torch.tensor(3.0)
    assert torch.equal(lm.dropout(s.cuda(), 0.25, 1, 2).cpu(), expected(s.view(1, 1), 0.25, 1, 2).view(()))


@pytest.mark.parametrize("shape", [(0, 8), (8, 0), (0,), (0, 0)])
def test_empty(lm, shape):
    assert lm.dropout(torch.empty(shape, device="cuda"), 0.5, 1, 1).shape == shape


def test_offsets_beyond_32_bits_of_elements(lm):
    """A column past 2^32 bytes and a row stride past 2^32 elements' bytes."""
    width = (1 << 30) + 24
    x = torch.ones(2, width, dtype=torch.float16, device="cuda")
    got = lm.dropout(x, 0.5, 9, 9)
    tail = got[1, -1000:].cpu()
    first = (width - 1000) // 8 * 8
    block = np.arange(first // 8, (width + 7) // 8, dtype=np.uint64)
    one = np.ones_like(block)
    words = ref.philox([block, one, one * np.uint64(9), one * np.uint64(0)], [9, 0])
    lanes = np.stack([w >> np.uint64(16 * i) & np.uint64(0xFFFF) for w in words for i in (0, 1)], 1).reshape(-1)
    lanes = lanes[width - 1000 - first:][:1000]
    assert torch.equal(tail, torch.from_numpy(np.where(lanes < 32768, 2.0, 0.0)).half())
    del x, got


def test_the_mask_is_made_again_for_the_gradient(lm):
    """dropout of the gradients with the same seed and offset is the backward pass; another offset is another
    mask; a device offset adds to the host's, modulo 2^64."""
    x = torch.randn(64, 1000, device="cuda")
    y = lm.dropout(x, 0.4, 7, 20)
    g = lm.dropout(torch.ones_like(x).to(torch.bfloat16), 0.4, 7, 20)
    assert torch.equal(y != 0, g != 0)
    assert not torch.equal(lm.dropout(x, 0.4, 7, 21) != 0, y != 0)
    assert not torch.equal(lm.dropout(x, 0.4, 8, 20) != 0, y != 0)
    more = torch.tensor([5], dtype=torch.int64, device="cuda")
    assert torch.equal(lm.dropout(x, 0.4, 7, 15, device_offset=more), y)
    assert torch.equal(lm.dropout(x, 0.4, 7, (1 << 64) - 5, device_offset=more + 20), y)


def test_share_of_dropped_elements(lm):
    """Binomial: 2^22 draws at p = 0.1 are within 6 standard deviations of the mean."""
    n = 1 << 22
    kept = int((lm.dropout(torch.ones(64, n // 64, device="cuda"), 0.1, 42, 0) != 0).sum())
    q = round(0.9 * 65536) / 65536
    assert abs(kept - n * q) < 6 * (n * q * (1 - q)) ** 0.5


def test_another_stream_and_a_recorded_graph(lm, gpu):
    x = torch.randn(128, 513, device="cuda")
    want = lm.dropout(x, 0.2, 1, 3)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    try:
        gpu.set_stream(side)
        got = lm.dropout(x, 0.2, 1, 3)  # torch's current stream is another: memory and kernel are side's
        side.synchronize()
        assert torch.equal(got, want)
        at = torch.zeros(1, dtype=torch.int64, device="cuda")
        out = torch.empty_like(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            lm.dropout(x, 0.2, 1, 3, device_offset=at, out=out)
            at.add_(1)
        for i in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out.cpu(), expected(x.cpu(), 0.2, 1, 3 + i))
    finally:
        torch.cuda.synchronize()
        gpu.set_stream(torch.cuda.current_stream())


def test_refusals(lm):
    from matrix_b200 import MtxcError, _abi

    x = torch.zeros(4, 8, device="cuda")
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(MtxcError) as e:
            lm.dropout(x, p, 0, 0)
        assert e.value.code == _abi.ERR_INVALID_ARGUMENT
    for bad in (x.to(torch.int32), x.to(torch.float64)):
        with pytest.raises(MtxcError) as e:
            lm.dropout(bad, 0.5, 0, 0)
        assert e.value.code == _abi.ERR_UNSUPPORTED_DTYPE
    with pytest.raises(ValueError, match="unit stride"):
        lm.dropout(x.t(), 0.5, 0, 0)
    with pytest.raises(ValueError, match="fold"):
        lm.dropout(torch.zeros(2, 6, 8, device="cuda")[:, :3], 0.5, 0, 0)
    with pytest.raises(ValueError, match="out"):
        lm.dropout(x, 0.5, 0, 0, out=torch.empty(4, 9, device="cuda"))
    with pytest.raises(ValueError, match="overlap"):
        lm.dropout(x, 0.5, 0, 0, out=torch.empty(8, device="cuda").expand(4, 8))
    with pytest.raises(ValueError, match="device_offset"):
        lm.dropout(x, 0.5, 0, 0, device_offset=torch.zeros(1, device="cuda"))
    lib = _abi.lib()
    state = _abi.DROPOUT_STATE.pack(0.5, 0, 0, 0)
    assert lib.mtxc_dropout(0, x.data_ptr(), None, 4, 8, 8, 8, state) == _abi.ERR_INVALID_ARGUMENT
    assert lib.mtxc_dropout(0, x.data_ptr(), x.data_ptr(), 4, 8, 8, 8, None) == _abi.ERR_INVALID_ARGUMENT
    assert lib.mtxc_dropout(0, x.data_ptr(), x.data_ptr(), 1 << 31, 8, 8, 8, state) == _abi.ERR_SHAPE


def test_outputs_written_in_place_are_noticed(lm):
    """autograd refuses to use a saved tensor that a call has written over since."""
    x = torch.ones(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    freq, pos = lm.rotary_frequencies(8)[0], torch.zeros(4, dtype=torch.int32, device="cuda")
    calls = {"dropout": lambda t: lm.dropout(t, 0.5, 0, 0, out=t), "residual": lambda t: lm.block_norm(t, x, out=t),
             "normed": lambda t: lm.block_norm(t, x, next_weight=w, normed_out=t),
             "rotary": lambda t: lm.rotary(t[:, None], None, pos, freq, out=(t[:, None], None)),
             "logits": lambda t: lm.logits_rules(t, out=t)}
    for name, call in calls.items():
        leaf = torch.ones(4, 8, device="cuda", requires_grad=True)
        saved = leaf * 1.5
        y = (saved * saved).sum()
        before = saved._version
        call(saved.detach())
        assert saved._version > before, name
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():  # tensors without a version
        t = torch.ones(4, 8, device="cuda")
        assert lm.dropout(t, 0.5, 0, 0, out=t) is t
