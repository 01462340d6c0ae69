"""The block norm and its backward pass (mtxc_block_norm, mtxc_block_norm_backward) against the formulas in 64
bits, within the bounds of tests/lm_reference.py."""
import pytest
import torch

from tests import lm_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-5
SEED, OFFSET = 0x1234567812345678, 1 << 40


@pytest.fixture
def lm(gpu):
    from matrix_b200 import lm

    return lm


class Case:
    """Inputs of one call on the host and the device; rows as `shape` minus its last axis."""

    def __init__(self, shape, dtype, gate=None, post=True, next=True, drop=0.0, alpha=1.0, beta=1.0, w0=0.0,
                 wdtype=None, gdtype=None, branch=True, seed=0):
        g = torch.Generator().manual_seed(seed + sum(shape))
        self.shape, self.width = shape, shape[-1]
        self.rows = 1
        for n in shape[:-1]:
            self.rows *= n
        wdtype, gdtype = wdtype or dtype, gdtype or dtype

        def normal(*s, mean=0.0, std=1.0, t=dtype):
            return (torch.randn(*s, generator=g) * std + mean).to(t)

        self.x = normal(*shape, std=2.0)
        self.b = normal(*shape, std=0.7) if branch else None
        self.dh, self.da = normal(*shape, std=0.3), normal(*shape, std=0.3) if next else None
        self.post = normal(self.width, mean=1.0 - w0, std=0.2, t=wdtype) if post and branch else None
        self.next = normal(self.width, mean=1.0 - w0, std=0.2, t=wdtype) if next else None
        gshape = {None: None, "channel": shape[-1:], "token": shape, "sequence": (shape[0],) + (1,) * (len(shape) - 2) + shape[-1:]}[gate]
        self.gate = normal(*gshape, mean=0.3, std=0.8, t=gdtype) if gshape and branch else None
        self.how = dict(residual_scale=alpha, branch_scale=beta, weight_offset=w0, dropout=drop, seed=SEED, offset=OFFSET)
        self.mask = ref.keep_mask(drop, SEED, OFFSET, self.rows, self.width) if drop else 1.0
        self.alpha, self.beta, self.w0 = (torch.tensor(v).double().item() for v in (alpha, beta, w0))
        groups = self.gate.numel() // self.width if self.gate is not None and self.width else 1
        self.gate_rows = max(1, self.rows // max(1, groups))

    def flat(self, t):
        return t.double().reshape(self.rows, self.width) if t is not None else None

    def cuda(self, t):
        return t.cuda() if t is not None else None

    def params(self):
        return dict(post_weight=self.cuda(self.post), gate=self.cuda(self.gate), next_weight=self.cuda(self.next), **self.how)

    def exact(self, x=None, b=None):
        d = lambda t: t.double() if t is not None else None  # noqa: E731
        g = self.gate.double().reshape(-1, self.width) if self.gate is not None else None
        x = self.flat(self.x) if x is None else x
        b = self.flat(self.b) if b is None else b
        eps = torch.tensor(EPS).double().item()  # as the call takes it, in 32 bits
        return ref.block_norm(x, b, d(self.post), g, self.gate_rows, d(self.next), self.alpha, self.beta, self.w0, eps, self.mask)

    def check_forward(self, lm, x=None, b=None, **more):
        o = lm.block_norm(self.cuda(self.x) if x is None else x, self.cuda(self.b) if b is None else b, eps=EPS,
                          **self.params(), **more)
        h, h_mag, a, a_mag, r, s = self.exact()
        what = f"{self.shape} {self.x.dtype}"
        ref.assert_within(o.residual.reshape(self.rows, self.width), h, h_mag, what + " residual")
        assert (o.normed is None) == (self.next is None)
        if a is not None:
            ref.assert_within(o.normed.reshape(self.rows, self.width), a, a_mag, what + " normed")
        if more.get("save_rstd", True):
            if r is not None:
                ref.assert_within(o.post_rstd, r, r, what + " post_rstd")
            if s is not None:
                share = h_mag.square().mean(1).sqrt() * s
                ref.assert_within(o.next_rstd, s, s * share, what + " next_rstd")
        return o

    def stored(self):
        """h as stored, and the rstds that go with the stored values, in 32 bits."""
        h = self.x  # any rows serve: the backward pass takes h as it is
        s = (self.flat(h).square().mean(1) + EPS).rsqrt().float() if self.next is not None else None
        r = (self.flat(self.b).square().mean(1) + EPS).rsqrt().float() if self.post is not None else None
        return h, r, s

    def check_backward(self, lm, dh=True, wrap=lambda t: t, **more):
        h, r, s = self.stored()
        dh = self.dh if dh else None
        up = lambda t: wrap(t.cuda()) if t is not None else None  # noqa: E731
        g = lm.block_norm_backward(up(dh), up(self.da), up(h), up(self.b), post_rstd=self.cuda(r), next_rstd=self.cuda(s),
                                   **self.params(), **more)
        d = lambda t: t.double() if t is not None else None  # noqa: E731
        gate = self.gate.double().reshape(-1, self.width) if self.gate is not None else None
        want = ref.block_norm_backward(self.flat(dh), self.flat(self.da), self.flat(h), self.flat(self.b), d(r), d(s),
                                       d(self.post), gate, self.gate_rows, d(self.next), self.alpha, self.beta, self.w0,
                                       self.mask)
        if not more.get("parameters", True):
            want = {k: v for k, v in want.items() if k in ("residual", "branch")}
        for name in g._fields:
            got = getattr(g, name)
            assert (got is not None) == (name in want), name
            if got is not None:
                ref.assert_within(got.reshape(want[name][0].shape), *want[name], f"{self.shape} {self.x.dtype} d_{name}")
        if g.gate is not None:
            assert g.gate.shape == self.gate.shape and g.gate.dtype == self.gate.dtype
        for w in (g.post_weight, g.next_weight):
            assert w is None or w.dtype == torch.float32
        return g


WIDTHS = [1, 2, 7, 8, 31, 33, 64, 100, 255, 256, 257, 512, 1000, 1024, 1032, 2001, 2048, 4096, 5000, 8192, 8200, 12288, 16384,
          16392, 20001, 32768, 40000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_forward_widths(lm, dtype, width):
    Case((5, width), dtype, gate="channel", drop=0.2, alpha=0.5, beta=1.25).check_forward(lm)
    Case((2, width), dtype).check_forward(lm)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_backward_widths(lm, dtype, width):
    Case((5, width), dtype, gate="channel", drop=0.2, alpha=0.5, beta=1.25).check_backward(lm)
    Case((2, width), dtype, gate="token").check_backward(lm)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [8193, 16385, 32776, 50001, 65536, 65544, 70001])
def test_backward_of_wide_rows(lm, dtype, width):
    """Rows shared by 2, 4 and 8 blocks, and rows past 65,536."""
    Case((7, width), dtype, gate="channel", drop=0.2, alpha=0.5).check_backward(lm)
    Case((3, 2, width), dtype, gate="sequence").check_backward(lm)
    Case((300, width // 8 + 8192), dtype).check_backward(lm)


@pytest.mark.parametrize("width", [64, 100, 2048, 2049])
@pytest.mark.parametrize("rows", [1, 3, 147, 149, 300, 1500])
def test_rows(lm, rows, width):
    for dtype in (torch.float32, torch.bfloat16):
        c = Case((rows, width), dtype, gate="channel", drop=0.1)
        c.check_forward(lm)
        c.check_backward(lm)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("next", [True, False])
@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token"])
@pytest.mark.parametrize("width", [96, 1001, 4096])
def test_parts(lm, dtype, post, next, gate, width):
    """Each norm and each kind of gate there or not."""
    c = Case((3, 5, width), dtype, gate=gate, post=post, next=next, drop=0.25 if next else 0.0)
    c.check_forward(lm)
    c.check_backward(lm)


@pytest.mark.parametrize("batch,length", [(1, 400), (2, 333), (400, 1), (400, 2), (7, 64), (290, 3), (1000, 2)])
@pytest.mark.parametrize("width", [72, 515, 1024])
def test_gradient_of_a_shared_gate(lm, batch, length, width):
    """More gate rows than blocks, fewer, and rows that blocks share: each sums over its own rows only."""
    for dtype in (torch.float32, torch.float16):
        Case((batch, length, width), dtype, gate="sequence").check_backward(lm)


def test_a_gate_per_outer_axis(lm):
    """[a, b, 1, width] on [a, b, c, width]: rows of two axes share, and the last group may be short."""
    c = Case((3, 4, 6, 80), torch.float32, gate=None)
    c.gate = torch.randn(3, 4, 1, 80)
    c.gate_rows = 6
    c.check_forward(lm)
    c.check_backward(lm)
    c.gate = torch.randn(3, 1, 1, 80)
    c.gate_rows = 24
    c.check_forward(lm)
    c.check_backward(lm)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width", [128, 999, 4096])
def test_float_weights_and_gate(lm, dtype, width):
    c = Case((9, width), dtype, gate="token", wdtype=torch.float32, gdtype=torch.float32, w0=1.0)
    c.check_forward(lm)
    c.check_backward(lm)
    c = Case((9, width), dtype, gate="channel", wdtype=torch.float32, w0=1.0)
    c.check_forward(lm)
    c.check_backward(lm)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [64, 1000, 2048])
def test_norm_alone(lm, dtype, width):
    """Without a branch: the norm in front of the first block; the residual goes through untouched."""
    c = Case((4, width), dtype, branch=False)
    x = c.x.cuda()
    o = lm.block_norm(x, eps=EPS, next_weight=c.next.cuda())
    assert o.residual is x and o.post_rstd is None
    h, _, a, a_mag, _, s = c.exact()
    ref.assert_within(o.normed, a, a_mag, "normed")
    ref.assert_within(o.next_rstd, s, s, "next_rstd")
    c.check_backward(lm)
    c.check_backward(lm, dh=False)
    scaled = lm.block_norm(x, residual_scale=0.25, eps=EPS)
    assert torch.equal(scaled.residual, x * 0.25) and scaled.normed is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,stride,start", [(64, 80, 0), (64, 67, 1), (1000, 1003, 5), (2048, 2056, 8), (4096, 4097, 3),
                                                (257, 258, 0), (8192, 8200, 16)])
def test_strides_and_alignment(lm, dtype, width, stride, start):
    c = Case((6, width), dtype, gate="token", drop=0.1)

    def view(t):
        base = torch.zeros(start + 6 * stride, dtype=dtype, device="cuda")
        v = torch.as_strided(base, (6, width), (stride, 1), start)
        return v.copy_(t.cuda())

    ends = [torch.as_strided(torch.full((start + 6 * stride,), 7.0, dtype=dtype, device="cuda"), (6, width), (stride, 1), start)
            for _ in range(2)]
    o = c.check_forward(lm, view(c.x), view(c.b), out=ends[0], normed_out=ends[1])
    assert o.residual is ends[0] and o.normed is ends[1]
    for e in ends:  # nothing outside the rows was written
        e.fill_(7.0)
        whole = torch.as_strided(e, (start + 6 * stride,), (1,), 0)
        assert torch.equal(whole, torch.full_like(whole, 7.0))
    c.check_backward(lm, wrap=lambda t: view(t))


@pytest.mark.parametrize("width", [100, 4096, 40000])
def test_in_place(lm, width):
    """The stream and the branch may be overwritten by the outputs."""
    c = Case((7, width), torch.bfloat16, gate="channel", drop=0.1)
    x, b = c.x.cuda(), c.b.cuda()
    want = lm.block_norm(c.x.cuda(), c.b.cuda(), eps=EPS, **c.params())
    o = lm.block_norm(x, b, eps=EPS, **c.params(), out=x, normed_out=b)
    assert o.residual is x and o.normed is b
    assert torch.equal(x, want.residual) and torch.equal(b, want.normed)


def test_serving_form_and_choices(lm):
    c = Case((1, 4096), torch.bfloat16)
    o = c.check_forward(lm, save_rstd=False)
    assert o.post_rstd is None and o.next_rstd is None
    c = Case((50, 512), torch.float32, gate="channel")
    c.check_backward(lm, parameters=False)
    c.check_backward(lm, dh=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [40, 1024, 8192])
def test_rows_of_zeros_and_special_values(lm, dtype, width):
    """A zero row stays finite (eps); a row with an infinity or NaN is not finite and leaves the others alone;
    everything dropped leaves the residual."""
    c = Case((5, width), dtype)
    c.x[0], c.b[0] = 0, 0
    c.check_forward(lm)
    c.check_backward(lm)
    x, b = c.x.clone(), c.b.clone()
    x[1, 3], b[2, 5] = float("inf"), float("nan")
    o = lm.block_norm(x.cuda(), b.cuda(), eps=EPS, **c.params())
    plain = lm.block_norm(c.x.cuda(), c.b.cuda(), eps=EPS, **c.params())
    for got, want in ((o.residual, plain.residual), (o.normed, plain.normed)):
        assert torch.equal(got[[0, 3, 4]], want[[0, 3, 4]])
    assert torch.isnan(o.normed[2]).all() and torch.isnan(o.normed[1, 3]) and torch.isinf(o.residual[1, 3])
    c.how["dropout"] = 1.0
    o = lm.block_norm(c.x.cuda(), b.cuda(), eps=EPS, **c.params())
    assert torch.equal(o.residual.cpu(), c.x)  # also where the branch is NaN: a dropped element is a zero


@pytest.mark.parametrize("shape", [(0, 64), (0, 3, 64), (4, 0)])
def test_empty(lm, shape):
    c = Case(shape, torch.float32, gate="channel")
    o = lm.block_norm(c.cuda(c.x), c.cuda(c.b), eps=EPS, **c.params())
    assert o.residual.shape == shape and o.normed.shape == shape
    rows = shape[0]
    z = torch.zeros(rows if shape[-1] == 0 else 0, device="cuda")
    if shape[-1]:
        g = lm.block_norm_backward(c.cuda(c.dh), c.cuda(c.da), c.cuda(c.x), c.cuda(c.b), post_rstd=z, next_rstd=z, **c.params())
        assert not g.post_weight.any() and not g.next_weight.any() and not g.gate.any()
        assert g.residual.shape == shape


def test_equal_calls_give_equal_bits(lm):
    c = Case((700, 1024), torch.bfloat16, gate="channel", drop=0.1)
    a, b = c.check_backward(lm), c.check_backward(lm)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_backward_mask_is_the_forward_one(lm):
    """With everything else 1, the gradient at the branch is nonzero exactly where the forward pass kept it."""
    x, b = torch.zeros(40, 333, device="cuda"), torch.ones(40, 333, device="cuda")
    how = dict(dropout=0.5, seed=4, offset=5)
    h = lm.block_norm(x, b, **how).residual
    g = lm.block_norm_backward(torch.ones_like(x), None, h, b, **how)
    assert torch.equal(h, g.branch) and torch.equal(h, lm.dropout(b, 0.5, 4, 5))


@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token"])
def test_gradients_against_differences(lm, gate):
    """The kernel's gradients (float32) against central differences of the forward formula in 64 bits: with
    steps of 1e-5 those are off by about 1e-10, so the bound is the arithmetic's."""
    c = Case((2, 3, 10), torch.float32, gate=gate, drop=0.25, alpha=0.75, beta=1.5)
    h, r, s = None, None, None
    o = lm.block_norm(c.x.cuda(), c.b.cuda(), eps=EPS, **c.params())
    g = lm.block_norm_backward(c.dh.cuda(), c.da.cuda(), o.residual, c.b.cuda(), post_rstd=o.post_rstd, next_rstd=o.next_rstd,
                               **c.params())
    eps = torch.tensor(EPS).double().item()
    named = {"residual": c.flat(c.x), "branch": c.flat(c.b), "post_weight": c.post.double(), "next_weight": c.next.double()}
    if gate:
        named["gate"] = c.gate.double().reshape(-1, 10)

    def loss(v):
        h, _, a, _, _, _ = ref.block_norm(v["residual"], v["branch"], v["post_weight"], v.get("gate"), c.gate_rows,
                                          v["next_weight"], c.alpha, c.beta, 0.0, eps, c.mask)
        return (h * c.flat(c.dh)).sum() + (a * c.flat(c.da)).sum()

    for name, t in named.items():
        got = getattr(g, name).double().cpu().reshape(-1)
        for i in range(t.numel()):
            vals = []
            for step in (1e-5, -1e-5):
                v = {k: u.clone() for k, u in named.items()}
                v[name].view(-1)[i] += step
                vals.append(loss(v))
            want = (vals[0] - vals[1]).item() / 2e-5
            # h is stored in 32 bits and enters every term: 2^-18 of the largest gradients of this size (~ 4)
            assert abs(got[i].item() - want) <= 2.0 ** -18 * (4 + abs(want)), (name, i, got[i].item(), want)


def test_many_rows_and_long_strides(lm):
    """Row offsets past 2^32 bytes, by a stride of 2^28 elements."""
    base = torch.zeros((9 << 28) + 64, dtype=torch.float16, device="cuda")
    x = torch.as_strided(base, (10, 64), (1 << 28, 1))
    c = Case((10, 64), torch.float16)
    x.copy_(c.x)
    c.check_forward(lm, x=x)
    c.check_backward(lm, wrap=lambda t: torch.as_strided(base, (10, 64), (1 << 28, 1)).copy_(t) if torch.equal(t.cpu(), c.x) else t)


def test_another_stream(lm, gpu):
    c = Case((64, 1024), torch.bfloat16, gate="channel")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    x, b = c.x.cuda(), c.b.cuda()
    want = lm.block_norm(x, b, eps=EPS, **c.params())
    torch.cuda.synchronize()
    try:
        gpu.set_stream(side)
        p = c.params()
        torch.cuda.synchronize()
        got = lm.block_norm(x, b, eps=EPS, **p)
        side.synchronize()
        assert torch.equal(got.residual, want.residual) and torch.equal(got.normed, want.normed)
    finally:
        torch.cuda.synchronize()
        gpu.set_stream(torch.cuda.current_stream())


def test_refusals(lm):
    from matrix_b200 import MtxcError, _abi

    x = torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for call in (lambda: lm.block_norm(x, x[:2]), lambda: lm.block_norm(x, x.half()), lambda: lm.block_norm(x, post_weight=w),
                 lambda: lm.block_norm(x, gate=w), lambda: lm.block_norm(x, x, post_weight=w[:4]),
                 lambda: lm.block_norm(x, x, post_weight=w, next_weight=w.half()), lambda: lm.block_norm(x.t(), x.t()),
                 lambda: lm.block_norm(x, x, gate=torch.ones(2, 8, device="cuda")),
                 lambda: lm.block_norm(x.view(2, 2, 8), x.view(2, 2, 8), gate=torch.ones(1, 2, 8, device="cuda")),
                 lambda: lm.block_norm(x, x, gate=torch.tensor(1.0, device="cuda")),
                 lambda: lm.block_norm(x, x, normed_out=x), lambda: lm.block_norm(x, x, out=x.half()),
                 lambda: lm.block_norm(x, x, post_weight=w.cpu()),
                 lambda: lm.block_norm_backward(x, x, x, x), lambda: lm.block_norm_backward(x, None, x, x, post_weight=w),
                 lambda: lm.block_norm_backward(x, x, x, x, next_weight=w, next_rstd=w[:2])):
        with pytest.raises(ValueError):
            call()
    i = x.to(torch.int32)
    for call, code in ((lambda: lm.block_norm(i, i), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.block_norm(x, x, post_weight=w.half()), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.block_norm(x, x, gate=w.to(torch.bfloat16)), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.block_norm(x, x, dropout=2.0), _abi.ERR_INVALID_ARGUMENT)):
        with pytest.raises(MtxcError) as e:
            call()
        assert e.value.code == code


@pytest.mark.parametrize("width", [64, 4096, 70000])
def test_gradients_in_place_and_of_a_scaled_stream(lm, gpu, width):
    """Through the C ABI: gradients written over the tensors they are made from; and without norm and branch, where
    the call needs no residual_out at all."""
    from matrix_b200 import _abi

    lib = _abi.lib()
    c = Case((6, width), torch.float32)
    h, r, s = c.stored()
    dh, da, b, hd = (t.cuda() for t in (c.dh, c.da, c.b, h))
    kept = [t.cuda() for t in (r, s, c.post, c.next)]
    want = lm.block_norm_backward(dh, da, hd, b, post_rstd=kept[0], next_rstd=kept[1], post_weight=kept[2],
                                  next_weight=kept[3], parameters=False)
    at = [t.data_ptr() for t in kept]
    drop = (0.0, 0, 0, 0)
    _abi.check(lib.mtxc_block_norm_backward(0, _abi.BLOCK_NORM_BACKWARD_ARGS.pack(
        6, width, dh.data_ptr(), width, da.data_ptr(), width, hd.data_ptr(), width, b.data_ptr(), width, *at, 0, 0, 0,
        dh.data_ptr(), width, b.data_ptr(), width, 0, 0, 0, 0, 0, 0, 1.0, 1.0, 0.0, *drop)))
    gpu.sync()
    assert torch.equal(dh, want.residual) and torch.equal(b, want.branch)
    dx = torch.empty_like(dh)
    _abi.check(lib.mtxc_block_norm_backward(0, _abi.BLOCK_NORM_BACKWARD_ARGS.pack(
        6, width, dh.data_ptr(), width, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, dx.data_ptr(), width, 0, 0, 0, 0, 0, 0, 0, 0,
        0.5, 1.0, 0.0, *drop)))
    gpu.sync()
    assert torch.equal(dx, dh * 0.5)


def test_workspace_refusal(lm, gpu):
    """Partial sums that do not fit the thread's workspace: refused, and nothing is written."""
    from matrix_b200 import MtxcError, _abi

    lib = _abi.lib()
    c = Case((8, 4096), torch.float32, gate="channel")
    ws = torch.empty(4096 * 3 * 4 - 256, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    _abi.check(lib.mtxc_set_workspace(ws.data_ptr(), ws.numel() // 256 * 256))
    try:
        with pytest.raises(MtxcError) as e:
            c.check_backward(lm)
        assert e.value.code == _abi.ERR_WORKSPACE
        c.check_backward(lm, parameters=False)
        small = torch.empty(4096 * 3 * 4 * 2, dtype=torch.uint8, device="cuda")
        _abi.check(lib.mtxc_set_workspace(small.data_ptr(), small.numel()))
        c.check_backward(lm)  # two blocks' worth
    finally:
        torch.cuda.synchronize()
        _abi.check(lib.mtxc_shutdown())
        gpu.init(0)


@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.bfloat16, 10)])
@pytest.mark.parametrize("rows,width", [(1, 4096), (300, 64), (7, 1000), (300, 4096), (300, 4097), (40, 8200), (40, 12001), (100, 70000)])
@pytest.mark.parametrize("over", ["branch", "residual"])
def test_gradients_written_over_a_gate_per_token(lm, gpu, dtype, code, rows, width, over):
    """Through the C ABI: a gate per token has the rows' shape, so that a gradient may be written over it.  The sums
    over rows take the gate as it was."""
    from matrix_b200 import _abi

    c = Case((rows, width), dtype, gate="token", drop=0.1)
    h, r, s = c.stored()
    dh, da, hd, b, gate = (t.cuda() for t in (c.dh, c.da, h, c.b, c.gate))
    kept = [t.cuda() for t in (r, s, c.post, c.next)]
    got = {"residual": torch.empty_like(hd), "branch": torch.empty_like(hd), over: gate, "gate": torch.empty_like(hd),
           "post_weight": torch.empty(width, device="cuda"), "next_weight": torch.empty(width, device="cuda")}
    at = lambda t: (t.data_ptr(), width)  # noqa: E731
    _abi.check(_abi.lib().mtxc_block_norm_backward(code, _abi.BLOCK_NORM_BACKWARD_ARGS.pack(
        rows, width, *at(dh), *at(da), *at(hd), *at(b), *(t.data_ptr() for t in kept), *at(gate), 1, *at(got["residual"]),
        *at(got["branch"]), got["post_weight"].data_ptr(), got["next_weight"].data_ptr(), *at(got["gate"]), code, code,
        1.0, 1.0, 0.0, 0.1, SEED, OFFSET, 0)))
    gpu.sync()
    want = ref.block_norm_backward(c.flat(c.dh), c.flat(c.da), c.flat(h), c.flat(c.b), r.double(), s.double(), c.post.double(),
                                   c.flat(c.gate), 1, c.next.double(), 1.0, 1.0, 0.0, c.mask)
    for name, (exact, magnitude) in want.items():
        ref.assert_within(got[name], exact, magnitude, f"{(rows, width)} {dtype} d_{name}")


class Scaled(Case):
    """Rows of any magnitude, the first of them zero; eps is a hundredth of their mean square."""

    def __init__(self, shape, dtype, scale, **more):
        super().__init__(shape, dtype, **more)
        self.x, self.b = (self.x.double() * scale).to(dtype), (self.b.double() * scale).to(dtype)
        self.x[0], self.b[0] = 0, 0
        self.eps = (0.1 * scale) ** 2

    def stored(self):
        r, s = ((self.flat(t).square().mean(1) + self.eps).rsqrt().float() for t in (self.b, self.x))
        return self.x, r, s


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale,widths", [(1e14, (64, 1000, 4096, 8200, 12001, 70000)), (1e-14, (64, 1000, 4096, 8200, 12001, 70000)),
                                          (1e16, (64, 1000, 4096)), (1e-17, (64, 1000, 4096))])
@pytest.mark.parametrize("gate", ["channel", "token"])
def test_gradients_of_very_large_and_very_small_rows(lm, dtype, scale, widths, gate):
    """Where the cube of a deviation passes the range of 32 bits, and the gradients do not."""
    for width in widths:
        Scaled((5, width), dtype, scale, gate=gate, drop=0.2).check_backward(lm)
        Scaled((5, width), dtype, scale, gate=gate).check_backward(lm, dh=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [64, 333, 1000, 4096, 8200, 12001, 70000])
@pytest.mark.parametrize("gate", [None, "channel", "token"])
def test_dropped_elements_hold_anything(lm, dtype, width, gate):
    """Where an element is dropped the branch and the gradient above it may be infinite or NaN: what is dropped is a
    zero in both directions.  (Without a norm of the branch, whose mean square every element enters.)"""
    c = Case((7, width), dtype, gate=gate, post=False, next=False, drop=0.5)
    gone = (c.mask == 0).view(c.shape)
    b, dh = c.b.clone(), c.dh.clone()
    b[gone] = torch.tensor([float("inf"), float("nan"), float("-inf")], dtype=dtype).repeat(b.numel())[:int(gone.sum())]
    want = lm.block_norm_backward(c.dh.cuda(), None, c.x.cuda(), c.b.cuda(), **c.params())
    got = lm.block_norm_backward(c.dh.cuda(), None, c.x.cuda(), b.cuda(), **c.params())
    assert torch.equal(got.branch, want.branch) and torch.equal(got.residual, want.residual)
    assert gate is None or torch.equal(got.gate, want.gate)
    dh[gone] = torch.tensor([float("nan"), float("inf")], dtype=dtype).repeat(b.numel())[:int(gone.sum())]
    got = lm.block_norm_backward(dh.cuda(), None, c.x.cuda(), b.cuda(), **c.params())
    assert torch.equal(got.branch, want.branch)
    assert gate is None or torch.equal(got.gate, want.gate)
    forward = [lm.block_norm(c.x.cuda(), t.cuda(), **c.params()).residual for t in (c.b, b)]
    assert torch.equal(*forward)


def test_calls_from_two_threads(lm, gpu):
    """Two threads with streams and workspaces of their own call one kernel with blocks of different shared memory:
    every call is accepted and every result is that of one thread by itself."""
    import threading

    from matrix_b200 import _abi

    lib, at = _abi.lib(), lambda t: (t.data_ptr(), 4096)  # noqa: E731
    jobs = []
    for rows in (100, 900):  # one team in a block, two
        c = Case((rows, 4096), torch.bfloat16)
        h, r, s = c.stored()
        t = [v.cuda() for v in (c.dh, c.da, h, c.b, r, s, c.post, c.next)]
        want = lm.block_norm_backward(*t[:4], post_rstd=t[4], next_rstd=t[5], post_weight=t[6], next_weight=t[7])
        got = [torch.empty_like(v) for v in (want.residual, want.branch, want.post_weight, want.next_weight)]
        args = _abi.BLOCK_NORM_BACKWARD_ARGS.pack(
            rows, 4096, *at(t[0]), *at(t[1]), *at(t[2]), *at(t[3]), *(v.data_ptr() for v in t[4:]), 0, 0, 0, *at(got[0]),
            *at(got[1]), got[2].data_ptr(), got[3].data_ptr(), 0, 0, 10, 10, 1.0, 1.0, 0.0, 0.0, 0, 0, 0)
        jobs.append((args, got, want, t))
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(2)

    def work(args):
        try:
            _abi.check(lib.mtxc_init(0))
            start.wait(60)
            for i in range(4000):
                _abi.check(lib.mtxc_block_norm_backward(10, args))
                if i % 200 == 199:
                    _abi.check(lib.mtxc_sync())
        except Exception as e:
            failed.append(str(e))
        finally:
            lib.mtxc_sync()
            lib.mtxc_shutdown()

    threads = [threading.Thread(target=work, args=(job[0],)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for _, got, want, _ in jobs:
        for g, w in zip(got, (want.residual, want.branch, want.post_weight, want.next_weight)):
            assert torch.equal(g, w)


def test_one_tensor_for_two_outputs_is_refused(lm):
    from matrix_b200 import MtxcError, _abi

    c = Case((4, 64), torch.float32)
    x, b, out = c.x.cuda(), c.b.cuda(), torch.empty(4, 64, device="cuda")
    with pytest.raises(MtxcError) as e:
        lm.block_norm(x, b, **c.params(), out=out, normed_out=out)
    assert e.value.code == _abi.ERR_INVALID_ARGUMENT
    h, r, s = (t.cuda() for t in c.stored())
    at = lambda t: (t.data_ptr(), 64)  # noqa: E731
    dh, da, post, next = c.dh.cuda(), c.da.cuda(), c.post.cuda(), c.next.cuda()
    sums = torch.empty(64, device="cuda")
    for gradients in ((*at(out), *at(out), 0, 0), (0, 0, 0, 0, sums.data_ptr(), sums.data_ptr())):
        assert _abi.lib().mtxc_block_norm_backward(0, _abi.BLOCK_NORM_BACKWARD_ARGS.pack(
            4, 64, *at(dh), *at(da), *at(h), *at(b), r.data_ptr(), s.data_ptr(), post.data_ptr(), next.data_ptr(), 0, 0, 0,
            *gradients, 0, 0, 0, 0, 1.0, 1.0, 0.0, 0.0, 0, 0, 0)) == _abi.ERR_INVALID_ARGUMENT


def test_backward_on_another_stream(lm, gpu):
    """The pass that uses the workspace and two launches, on a stream of the caller's."""
    c = Case((640, 1024), torch.bfloat16, gate="channel", drop=0.1)
    h, r, s = (t.cuda() for t in c.stored())
    dh, da, b, p = c.dh.cuda(), c.da.cuda(), c.b.cuda(), c.params()
    call = lambda: lm.block_norm_backward(dh, da, h, b, post_rstd=r, next_rstd=s, **p)  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    try:
        gpu.set_stream(side)
        got = call()
        side.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    finally:
        torch.cuda.synchronize()
        gpu.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("rows,width", [(1, 4096), (300, 64), (7, 1000), (300, 4096), (300, 4097), (40, 12001)])
@pytest.mark.parametrize("over", ["branch", "residual"])
def test_gradients_written_over_a_gate_without_the_post_weight_s(lm, gpu, rows, width, over):
    """The same where no sum over rows needs the gate: the bits are those of separate tensors."""
    from matrix_b200 import _abi

    c = Case((rows, width), torch.bfloat16, gate="token", drop=0.1)
    h, r, s = c.stored()
    dh, da, hd, b, gate = (t.cuda() for t in (c.dh, c.da, h, c.b, c.gate))
    kept = [t.cuda() for t in (r, s, c.post, c.next)]
    want = lm.block_norm_backward(dh, da, hd, b, post_rstd=kept[0], next_rstd=kept[1], **c.params())
    got = {"residual": torch.empty_like(hd), "branch": torch.empty_like(hd), over: gate, "gate": torch.empty_like(hd),
           "next_weight": torch.empty(width, device="cuda")}
    at = lambda t: (t.data_ptr(), width)  # noqa: E731
    _abi.check(_abi.lib().mtxc_block_norm_backward(10, _abi.BLOCK_NORM_BACKWARD_ARGS.pack(
        rows, width, *at(dh), *at(da), *at(hd), *at(b), *(t.data_ptr() for t in kept), *at(gate), 1, *at(got["residual"]),
        *at(got["branch"]), 0, got["next_weight"].data_ptr(), *at(got["gate"]), 10, 10, 1.0, 1.0, 0.0, 0.1, SEED, OFFSET, 0)))
    gpu.sync()
    for name, t in got.items():
        assert torch.equal(t, getattr(want, name)), name
