"""Head norms with rotary positions (mtxc_head_norm_rotary and its backward pass) against the formulas in 64 bits.

The bound: a result is rounded once, by 2^-p of itself; before that sums of a head in 32 bits (less than 48 * 2^-24 of the
magnitudes), a square root, the angle (2^-20, as rotary's own tests derive it) and about ten products: within 2^-18 of the
formula's magnitude.  The angle, up to four roundings in 64 bits, adds 2^-51 of itself."""
import threading

import pytest
import torch

from tests import attention_reference as att
from tests import lm_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture
def lm(gpu):
    from matrix_b200 import lm

    return lm


def normal(*shape, dtype=torch.float32, seed=0, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape))
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype)


def check(lm, q, k, positions, f, wq=None, wk=None, w0=0.0, eps=1e-6, scale=1.0, interleaved=False, parameters=True, seed=5):
    """q, k: device tensors [batch, length, heads, head] (k may be None): forward and backward."""
    how = dict(q_weight=None if wq is None else wq.cuda(), k_weight=None if wk is None else wk.cuda(), weight_offset=w0,
               scale=scale, interleaved=interleaved)
    pos, fd = positions.cuda(), f.cuda()
    o = lm.head_norm_rotary(q, k, pos, fd, eps=eps, **how)
    s = torch.tensor(scale).double().item()
    dy = [None if x is None else normal(*x.shape, dtype=x.dtype, seed=seed, std=0.3).cuda() for x in (q, k)]
    g = lm.head_norm_rotary_backward(*dy, q, k, pos, fd, q_rstd=o.q_rstd, k_rstd=o.k_rstd, parameters=parameters, **how)
    angle = positions.double().abs().max().item() * (f.max().item() if len(f) else 0.0) if positions.numel() else 0.0
    work = ref.WORK + 2.0 ** -51 * angle
    for x, w, y, rstd, d, dx, dw, name in ((q, wq, o.q, o.q_rstd, dy[0], g.q, g.q_weight, "q"),
                                           (k, wk, o.k, o.k_rstd, dy[1], g.k, g.k_weight, "k")):
        if x is None:
            assert y is None and rstd is None and dx is None and dw is None
            continue
        what = f"{name} {tuple(x.shape)} {x.dtype} part {2 * len(f)}"
        x64, w64 = x.cpu().double(), None if w is None else w.double()
        want, mag, r = att.head_norm(x64, w64, w0, torch.tensor(eps).double().item(), positions, f, s, interleaved)
        ref.assert_within(y, want, mag, what, work)
        ref.assert_within(rstd, r, r, what)
        back = att.head_norm_backward(d.cpu().double(), x64, w64, w0, rstd.cpu().double(), positions, f, s, interleaved)
        ref.assert_within(dx, *back["x"], what + " gradient", work)
        if w is None or not parameters:
            assert dw is None
        else:
            assert dw.dtype == torch.float32
            ref.assert_within(dw, *back["weight"], what + " weight's gradient", work)
    return o, g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head,part", [(1, 0), (2, 2), (3, 2), (8, 8), (16, 6), (64, 64), (65, 64), (80, 32), (80, 80), (96, 96),
                                       (100, 50), (128, 128), (128, 64), (128, 0), (192, 64), (256, 256), (512, 512), (1024, 1024),
                                       (1000, 600)])
def test_heads_and_parts(lm, dtype, interleaved, head, part):
    f = lm.rotary_frequencies(part, device="cpu")[0]
    wq, wk = normal(head, mean=1.0, std=0.2, dtype=dtype), normal(head, mean=1.0, std=0.2, dtype=dtype, seed=1)
    for batch, length, qh, kh in ((1, 1, 1, 1), (2, 5, 6, 2), (3, 17, 7, 1), (2, 9, 4, 0)):
        q = normal(batch, length, qh, head, dtype=dtype, std=2.0).cuda()
        k = normal(batch, length, kh, head, dtype=dtype, seed=1).cuda() if kh else None
        positions = torch.randint(0, 4096, (batch, length), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
        check(lm, q, k, positions, f, wq, wk if kh else None, interleaved=interleaved)
    check(lm, q, None, positions, f, None, None, scale=1.25, interleaved=interleaved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weight_dtype", TYPES)
@pytest.mark.parametrize("head", [64, 80, 66])
def test_weights(lm, dtype, weight_dtype, head):
    """Of every type, of one side only, with an offset, not wanted."""
    f = lm.rotary_frequencies(64, device="cpu")[0]
    q, k = normal(2, 33, 5, head, dtype=dtype).cuda(), normal(2, 33, 3, head, dtype=dtype, seed=3).cuda()
    positions = torch.arange(33, dtype=torch.int64)[None].expand(2, 33)
    w = normal(head, dtype=weight_dtype, std=0.2)
    check(lm, q, k, positions, f, w, None, w0=1.0)
    check(lm, q, k, positions, f, None, w, w0=1.0)
    check(lm, q, k, positions, f, w, w, w0=1.0, parameters=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,length,qh,kh,head", [(1, 1, 32, 8, 128), (64, 1, 32, 8, 128), (2, 1023, 7, 1, 80), (3, 700, 16, 16, 64),
                                                     (1, 4099, 3, 2, 96), (1, 300, 1, 130, 64), (1, 40, 300, 1, 128)])
def test_sizes(lm, dtype, interleaved, batch, length, qh, kh, head):
    """From a decode step to several tiles of a block, more heads than a block takes at a time."""
    f, scale = lm.rotary_frequencies(head, 500000.0, scaling="by_parts", factor=32, original_length=8192, device="cpu")
    q, k = normal(batch, length, qh, head, dtype=dtype).cuda(), normal(batch, length, kh, head, dtype=dtype, seed=2).cuda()
    positions = torch.randint(0, 131072, (batch, length), generator=torch.Generator().manual_seed(2))
    w = normal(head, mean=1.0, std=0.1, dtype=dtype)
    check(lm, q, k, positions, f, w, w, scale=scale, interleaved=interleaved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts(lm, dtype, interleaved):
    """Heads before tokens, slices of one tensor of queries, keys and values, misaligned bases, one head for all,
    strided positions, three axes."""
    f = lm.rotary_frequencies(64, device="cpu")[0]
    positions = torch.arange(12, dtype=torch.int32).view(1, 12).expand(2, 12) + 100
    q = normal(2, 6, 12, 64, dtype=dtype).cuda().transpose(1, 2)
    k = normal(2, 2, 12, 64, dtype=dtype).cuda().transpose(1, 2)
    w = normal(64, mean=1.0, std=0.1, dtype=dtype)
    o, _ = check(lm, q, k, positions, f, w, w, interleaved=interleaved)
    assert o.q.stride() == q.stride() and o.q_rstd.is_contiguous()
    for head in (64, 70, 65):
        qkv = normal(2, 12, 10, head, dtype=dtype).cuda()
        wh = normal(head, mean=1.0, std=0.1, dtype=dtype)
        check(lm, qkv[:, :, :6], qkv[:, :, 6:8], positions, f, wh, wh, interleaved=interleaved)
    for start in (1, 3, 4, 8):
        base = normal(start + 2 * 12 * 6 * 72, dtype=dtype).cuda()
        check(lm, torch.as_strided(base, (2, 12, 6, 64), (12 * 6 * 72, 6 * 72, 72, 1), start), None, positions, f, w,
              interleaved=interleaved)
    one = normal(2, 12, 1, 64, dtype=dtype).cuda().expand(2, 12, 4, 64)
    check(lm, one, one[:, :, :2], positions, f, w, w, interleaved=interleaved)
    wide = torch.stack([positions, positions + 1], -1)
    a = lm.head_norm_rotary(q, k, wide.cuda()[..., 0], f.cuda(), q_weight=w.cuda(), interleaved=interleaved)
    b = lm.head_norm_rotary(q, k, positions.cuda(), f.cuda(), q_weight=w.cuda(), interleaved=interleaved)
    assert torch.equal(a.q, b.q) and torch.equal(a.k, b.k)
    c = lm.head_norm_rotary(q[1], k[1], positions[1].cuda(), f.cuda(), q_weight=w.cuda(), interleaved=interleaved)
    assert torch.equal(c.q, b.q[1]) and torch.equal(c.k_rstd, b.k_rstd[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head,part", [(64, 64), (64, 32), (67, 32)])
def test_in_place(lm, dtype, interleaved, head, part):
    f = lm.rotary_frequencies(part)[0]
    positions = torch.arange(7, dtype=torch.int32, device="cuda")
    qkv = normal(1, 7, 9, head, dtype=dtype).cuda()
    w = normal(head, mean=1.0, dtype=dtype).cuda()
    want = qkv.clone()
    o = lm.head_norm_rotary(qkv[:, :, :5], qkv[:, :, 5:7], positions, f, q_weight=w, interleaved=interleaved)
    want[:, :, :5], want[:, :, 5:7] = o.q, o.k
    views = qkv[:, :, :5], qkv[:, :, 5:7]
    version = qkv._version
    got = lm.head_norm_rotary(*views, positions, f, q_weight=w, interleaved=interleaved, out=views)
    assert got.q is views[0] and torch.equal(qkv, want) and qkv._version > version


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(lm, interleaved):
    f, scale = lm.rotary_frequencies(24, scaling="by_parts", factor=4, original_length=100, device="cpu")
    positions = torch.randint(0, 1000, (2, 3), generator=torch.Generator().manual_seed(0), dtype=torch.int32)
    x, w, dy = normal(2, 3, 2, 30), normal(30, mean=1.0, std=0.2), normal(2, 3, 2, 30, seed=9)
    s = torch.tensor(scale).double().item()
    how = dict(q_weight=w.cuda(), scale=scale, interleaved=interleaved)
    o = lm.head_norm_rotary(x.cuda(), None, positions.cuda(), f.cuda(), eps=1e-3, **how)
    g = lm.head_norm_rotary_backward(dy.cuda(), None, x.cuda(), None, positions.cuda(), f.cuda(), q_rstd=o.q_rstd, **how)

    def value(x, w):
        return (att.head_norm(x, w, 0.0, 1e-3, positions, f, s, interleaved)[0] * dy.double()).sum().item()

    # central differences of a step of 1e-4 in 64 bits: off by 1e-8 / 6 of third derivatives (below 1e3 here), 1e-11 of rounding
    back = att.head_norm_backward(dy.double(), x.double(), w.double(), 0.0, o.q_rstd.cpu().double(), positions, f, s, interleaved)
    for at, step, got, mag in ((0, 1e-4, g.q, back["x"][1]), (1, 1e-4, g.q_weight, back["weight"][1])):
        for i in range(0, (x, w)[at].numel(), 7):
            ends = []
            for sign in (1, -1):
                v = [x.double().clone(), w.double().clone()]
                v[at].view(-1)[i] += sign * step
                ends.append(value(*v))
            want = (ends[0] - ends[1]) / (2 * step)
            assert abs(got.view(-1)[i].item() - want) <= 2 * ref.WORK * mag.reshape(-1)[i].item() + 1e-5


def test_special_values_stay_in_their_head(lm):
    f = lm.rotary_frequencies(64)[0]
    x = normal(1, 4, 3, 64)
    x[0, 1, 0, 5], x[0, 2, 1, 40], x[0, 3, 2] = float("nan"), float("inf"), 0.0
    o = lm.head_norm_rotary(x.cuda(), None, torch.arange(4, dtype=torch.int32).cuda(), f)
    y = o.q.cpu()
    bad = torch.zeros(1, 4, 3, dtype=torch.bool)
    bad[0, 1, 0] = bad[0, 2, 1] = True
    assert torch.isfinite(y[~bad]).all() and torch.isnan(y[0, 1, 0]).all() and not torch.isfinite(y[0, 2, 1]).all()
    assert (y[0, 3, 2] == 0).all() and o.q_rstd[0, 3, 2].item() == pytest.approx(1000.0, rel=1e-6)


@pytest.mark.parametrize("shape", [(0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64), (2, 4, 3, 0)])
def test_empty(lm, shape):
    x = torch.empty(shape, device="cuda")
    w = torch.ones(shape[-1], device="cuda")
    positions = torch.zeros(shape[1], dtype=torch.int32, device="cuda")
    f = lm.rotary_frequencies(min(64, shape[-1]))[0]
    o = lm.head_norm_rotary(x, None, positions, f, q_weight=w)
    assert o.q.shape == shape and o.q_rstd.shape == shape[:-1]
    g = lm.head_norm_rotary_backward(x, None, x, None, positions, f, q_rstd=o.q_rstd, q_weight=w)
    assert g.q.shape == shape and (g.q_weight == 0).all()  # a sum over nothing


def test_equal_calls_give_equal_bits_and_streams(lm, gpu):
    """The partial sums come from the call's own memory: two streams do not disturb each other, nor two graphs."""
    from matrix_b200 import backend

    f = lm.rotary_frequencies(128)[0]
    cases = [(normal(1, 2048, 8, 128, seed=i).cuda(), normal(1, 2048, 8, 128, seed=i + 9).cuda()) for i in range(2)]
    positions = torch.arange(2048, dtype=torch.int32, device="cuda")
    w = normal(128, mean=1.0).cuda()

    def run(x, dy):
        o = lm.head_norm_rotary(x, None, positions, f, q_weight=w)
        return lm.head_norm_rotary_backward(dy, None, x, None, positions, f, q_rstd=o.q_rstd, q_weight=w)

    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    streams, graphs, got = [torch.cuda.Stream() for _ in cases], [], []
    try:
        for s, c in zip(streams, cases):
            backend.set_stream(s)
            with torch.cuda.stream(s):
                run(*c)
                s.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=s):
                    got.append(run(*c))
                graphs.append(graph)
        for _ in range(5):
            for g in got:
                for t in (g.q, g.q_weight):
                    t.zero_()
            torch.cuda.synchronize()
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a.q, b.q) and torch.equal(a.q_weight, b.q_weight)
    finally:
        backend.set_stream(torch.cuda.default_stream())


def test_threads(lm, gpu):
    """Two threads with streams of their own."""
    from matrix_b200 import backend

    f = lm.rotary_frequencies(128)[0]
    positions = torch.arange(500, dtype=torch.int32, device="cuda")
    cases = [(normal(1, 500, 8, 128, dtype=t).cuda(), normal(1, 500, 8, 128, dtype=t, seed=4).cuda(), normal(128, dtype=t).cuda())
             for t in (torch.float32, torch.bfloat16)]

    def run(x, dy, w):
        o = lm.head_norm_rotary(x, None, positions, f, q_weight=w)
        return lm.head_norm_rotary_backward(dy, None, x, None, positions, f, q_rstd=o.q_rstd, q_weight=w)

    want = [run(*c) for c in cases]
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
                    g = run(*cases[i])
                    s.synchronize()
                    if not (torch.equal(g.q, want[i].q) and torch.equal(g.q_weight, want[i].q_weight)):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
