"""The rules on logits (mtxc_logits_rules) against a token-by-token implementation in 64 bits.

The bound: at most five roundings in 32 bits, each of at most 2^-24 of the terms' magnitudes, which
tests/lm_reference.py adds up after the repetition rule: 2^-21 of them."""
import pytest
import torch

from tests import lm_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
WORK = 2.0 ** -21
INF = float("inf")


@pytest.fixture
def lm(gpu):
    from matrix_b200 import lm

    return lm


def inputs(rows, vocab, history, biases, seed=0, mask=True, padding=True):
    g = torch.Generator().manual_seed(seed + rows + vocab + history)

    def some(*shape):
        t = (torch.rand(*shape, generator=g).pow(3) * vocab).to(torch.int32).clamp_(max=vocab - 1)
        if padding and t.numel() > 4:  # entries that name no token
            t.view(-1)[1::5] = torch.tensor([-1, vocab, 2 ** 31 - 1, -2 ** 31]).to(torch.int32).repeat(t.numel())[:len(t.view(-1)[1::5])]
        return t

    d = dict(tokens=some(rows, history), lengths=torch.randint(0, history + 1, (rows,), generator=g, dtype=torch.int32),
             prompt_lengths=torch.randint(0, history // 2 + 1, (rows,), generator=g, dtype=torch.int32),
             repetition=torch.rand(rows, generator=g) + 0.7, frequency=torch.randn(rows, generator=g),
             presence=torch.randn(rows, generator=g), bias_tokens=some(rows, biases),
             bias_values=torch.randn(rows, biases, generator=g) * 5)
    if mask:
        d["mask"] = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=g).to(torch.int32)
    return d


def check(lm, logits, d, what="", **more):
    """logits: a device tensor; d: host tensors."""
    rows = logits.shape[0]
    got = lm.logits_rules(logits, **{k: v.cuda() for k, v in d.items()}, **more)
    lists = {}
    for k, v in d.items():
        v = v.expand(rows, v.shape[-1]) if k in ("tokens", "bias_tokens", "bias_values", "mask") else v
        lists[k] = v.tolist() if v.dtype == torch.int32 else v.double().tolist()
    want, mag = ref.logits_rules(logits.detach().cpu().double(), **lists)
    ref.assert_within(got, want, mag, f"{what} {tuple(logits.shape)} {logits.dtype}", WORK)
    return got


def normal(rows, vocab, dtype, std=3.0):
    return (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab)) * std).to(dtype).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 100, 1000, 4095, 4096, 4097, 8200, 12289, 50257])
def test_vocabularies(lm, dtype, vocab):
    check(lm, normal(3, vocab, dtype), inputs(3, vocab, 50, 9))


@pytest.mark.parametrize("rows,history,biases", [(1, 1, 1), (1, 3000, 300), (40, 17, 2), (700, 5, 3), (2, 4097, 1),
                                                 (2, 40000, 1), (3, 5, 2500)])
def test_rows_and_lists(lm, rows, history, biases):
    check(lm, normal(rows, 500, torch.float32), inputs(rows, 500, history, biases))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("keys", [(), ("repetition",), ("frequency",), ("presence",), ("frequency", "presence"), ("bias",), ("mask",),
                                  ("repetition", "mask"), ("repetition", "frequency", "presence", "bias", "mask")])
@pytest.mark.parametrize("told", ["all", "lengths", "both"])
def test_each_rule_alone(lm, dtype, keys, told):
    d = inputs(4, 777, 60, 12)
    use = {k for key in keys for k in (("bias_tokens", "bias_values") if key == "bias" else (key,))}
    if use & {"repetition", "frequency", "presence"}:
        use |= {"tokens"} | ({"lengths"} if told != "all" else set()) | ({"prompt_lengths"} if told == "both" else set())
    check(lm, normal(4, 777, dtype), {k: v for k, v in d.items() if k in use}, f"{keys} {told}")


def test_lengths_outside_the_list_are_cut(lm):
    d = inputs(5, 300, 20, 3)
    d["lengths"] = torch.tensor([-5, 0, 20, 21, 2 ** 31 - 1], dtype=torch.int32)
    d["prompt_lengths"] = torch.tensor([3, -1, 2 ** 31 - 1, -2 ** 31, 4], dtype=torch.int32)
    want = dict(d, lengths=d["lengths"].clamp(0, 20), prompt_lengths=d["prompt_lengths"].clamp(0, 20))
    a = check(lm, normal(5, 300, torch.float32), want)
    assert torch.equal(lm.logits_rules(normal(5, 300, torch.float32), **{k: v.cuda() for k, v in d.items()}), a)


def test_the_same_token_over_and_over(lm):
    """A count of thousands, in the prompt and generated; of several biases the last counts."""
    d = inputs(2, 64, 5000, 40, padding=False, mask=False)
    d["tokens"][:] = 7
    d["lengths"][:], d["prompt_lengths"][:] = 5000, torch.tensor([0, 4999])
    d["bias_tokens"][:] = 9
    y = check(lm, normal(2, 64, torch.float32), d)
    x = normal(2, 64, torch.float32)
    assert torch.equal(y[:, 9].cpu(), x[:, 9].cpu() + d["bias_values"][:, -1])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_without_an_allowed_token(lm, dtype):
    d = inputs(3, 1000, 30, 5)
    d["mask"][1] = 0
    y = check(lm, normal(3, 1000, dtype), d)
    assert torch.isneginf(y[1]).all() and torch.isfinite(y[0]).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_special_values(lm, dtype):
    """Infinities, NaN and the type's lowest value: masked ones are -inf like any other, the rest follow the rules."""
    d = inputs(2, 64, 30, 1, padding=False)
    d["tokens"] = torch.arange(30, dtype=torch.int32).expand(2, 30).contiguous()
    d["lengths"][:], d["prompt_lengths"][:] = 30, 10
    d["mask"][0], d["mask"][1] = -1, 0x55555555
    x = normal(2, 64, dtype)
    lowest = torch.finfo(dtype).min
    x[:, 0:8] = torch.tensor([INF, -INF, float("nan"), lowest, INF, -INF, float("nan"), lowest], dtype=dtype)
    x[:, 40:44] = torch.tensor([INF, -INF, float("nan"), lowest], dtype=dtype)
    y = lm.logits_rules(x, **{k: v.cuda() for k, v in d.items()})
    ok = torch.ones(64, dtype=torch.bool)
    ok[[2, 3, 6, 7, 42, 43]] = False
    want, mag = ref.logits_rules(x[:, ok].cpu().double(), mask=None)
    assert torch.isnan(y[0, [2, 6, 42]]).all()
    assert y[0, 43].item() == lowest or d["bias_tokens"][0, 0] == 43  # untouched
    odd = torch.arange(64) % 2 == 1
    assert torch.isneginf(y[1][odd]).all() and not torch.isneginf(y[1, 42])
    assert y[0, 0] == INF and y[0, 40] == INF and torch.isneginf(y[0, 1]) and torch.isneginf(y[0, 41])
    assert torch.isnan(y[1, 2]) and torch.isnan(y[1, 42])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,stride,start", [(1000, 1024, 0), (1000, 1001, 3), (4096, 4100, 4), (5000, 5000, 1)])
def test_strides_shared_lists_and_in_place(lm, dtype, vocab, stride, start):
    rows = 4
    base = torch.full((start + rows * stride,), 7.0, dtype=dtype, device="cuda")
    x = torch.as_strided(base, (rows, vocab), (stride, 1), start)
    x.copy_(normal(rows, vocab, dtype))
    d = inputs(rows, vocab, 33, 6)
    d["bias_tokens"], d["bias_values"], d["mask"] = d["bias_tokens"][0], d["bias_values"][:1], d["mask"][0]
    y = check(lm, x, d)
    x.copy_(normal(rows, vocab, dtype))
    got = lm.logits_rules(x, **{k: v.cuda() for k, v in d.items()}, out=x)
    assert got is x and torch.equal(x, y)
    x.fill_(7.0)
    assert torch.equal(base, torch.full_like(base, 7.0))  # nothing outside the rows was written
    wide = torch.zeros(rows, 50, dtype=torch.int32, device="cuda")
    wide[:, :33] = d["tokens"].cuda()
    a = lm.logits_rules(normal(rows, vocab, dtype), tokens=wide[:, :33], presence=d["presence"].cuda())
    b = lm.logits_rules(normal(rows, vocab, dtype), tokens=d["tokens"].cuda(), presence=d["presence"].cuda())
    assert torch.equal(a, b)


@pytest.mark.parametrize("shape", [(0, 8), (3, 0)])
def test_empty(lm, shape):
    assert lm.logits_rules(torch.empty(shape, device="cuda")).shape == shape


def test_empty_lists(lm):
    x = normal(2, 100, torch.float32)
    none = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    y = lm.logits_rules(x, tokens=none, repetition=torch.ones(2, device="cuda") * 2, bias_tokens=none, bias_values=none.float())
    assert torch.equal(x, y)


def test_long_offsets(lm):
    """Rows further than 2^32 bytes apart."""
    base = torch.zeros((2 << 30) + 4096, dtype=torch.float16, device="cuda")
    x = torch.as_strided(base, (3, 4096), (1 << 30, 1))
    x.copy_(normal(3, 4096, torch.float16))
    check(lm, x, inputs(3, 4096, 20, 3))


def test_the_choice_that_follows(lm, gpu):
    """A decode step's tail: the rules, then the framework's softmax and ArgMax on the same stream."""
    d = inputs(8, 4096, 100, 8)
    y = lm.logits_rules(normal(8, 4096, torch.float32), **{k: v.cuda() for k, v in d.items()})
    best = gpu.reduce("argmax", y, 1)
    p = gpu.softmax_lastdim(y)
    gpu.sync()
    assert torch.equal(best.cpu().long(), y.cpu().argmax(1))
    assert torch.equal(p.cpu() == 0, torch.isneginf(y).cpu() | (p.cpu() == 0)) and torch.allclose(p.sum(1).cpu(), torch.ones(8))


def test_another_stream(lm, gpu):
    d = {k: v.cuda() for k, v in inputs(8, 9000, 100, 8).items()}
    x = normal(8, 9000, torch.bfloat16)
    want = lm.logits_rules(x, **d)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    try:
        gpu.set_stream(side)
        got = lm.logits_rules(x, **d)
        side.synchronize()
        assert torch.equal(got, want)
    finally:
        torch.cuda.synchronize()
        gpu.set_stream(torch.cuda.current_stream())


def test_refusals(lm):
    from matrix_b200 import MtxcError, _abi

    x = torch.zeros(4, 64, device="cuda")
    t = torch.zeros(4, 5, dtype=torch.int32, device="cuda")
    r = torch.ones(4, device="cuda")
    m = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    for call in (lambda: lm.logits_rules(x[0]), lambda: lm.logits_rules(x, repetition=r), lambda: lm.logits_rules(x, tokens=t.long()),
                 lambda: lm.logits_rules(x, tokens=t[:3], repetition=r), lambda: lm.logits_rules(x, tokens=t, repetition=r[:3]),
                 lambda: lm.logits_rules(x, tokens=t, repetition=r.half()), lambda: lm.logits_rules(x, bias_tokens=t),
                 lambda: lm.logits_rules(x, bias_tokens=t, bias_values=t[:, :4].float()), lambda: lm.logits_rules(x, mask=m[:, :1]),
                 lambda: lm.logits_rules(x, mask=m.long()), lambda: lm.logits_rules(x, mask=m.cpu()),
                 lambda: lm.logits_rules(x.t()), lambda: lm.logits_rules(x, out=x[:2])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(MtxcError) as e:
        lm.logits_rules(x.int())
    assert e.value.code == _abi.ERR_UNSUPPORTED_DTYPE


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [64, 77])
def test_special_values_under_every_rule(lm, dtype, vocab):
    """Infinities, NaN and the type's lowest value, in the history, biased, masked and none of these: every element
    of the row is the formula's."""
    d = inputs(3, vocab, 30, 4, padding=False)
    d["tokens"] = torch.arange(30, dtype=torch.int32).expand(3, 30).contiguous()
    d["lengths"][:], d["prompt_lengths"][:] = 30, torch.tensor([10, 0, 30])
    d["bias_tokens"] = torch.tensor([[2, 3, 40, 43]], dtype=torch.int32).expand(3, 4).contiguous()
    d["mask"][0], d["mask"][1], d["mask"][2] = -1, 0x55555555, 0
    x = normal(3, vocab, dtype)
    lowest = torch.finfo(dtype).min
    x[:, 0:8] = torch.tensor([INF, -INF, float("nan"), lowest, INF, -INF, float("nan"), lowest], dtype=dtype)
    x[:, 40:44] = torch.tensor([INF, -INF, float("nan"), lowest], dtype=dtype)
    check(lm, x, d)
    check(lm, x, {k: v for k, v in d.items() if k != "mask"})
