"""Outputs that lie over what a call reads: the documented ones give what a call with outputs of its own gives, the others are
refused before anything runs (through the C ABI: the Python module makes gradients of its own)."""
import pytest
import torch

from matrix_b200 import MtxcError, _abi

pytestmark = pytest.mark.gpu

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 10}


@pytest.fixture
def lm(gpu):
    from matrix_b200 import lm

    return lm


def packed(fields, layout, values):
    """The struct's bytes: tensors as addresses, what is not given as zeros."""
    flat = []
    for field in fields:
        name, kind = field.split(":")
        n = int(kind[:-1] or 1)
        v = values.get(name, [0] * n)
        v = list(v) if isinstance(v, (list, tuple)) else [v]
        assert len(v) == n, name
        flat += [0 if x is None else x.data_ptr() if torch.is_tensor(x) else x for x in v]
    return layout.pack(*flat)


def strides(*tensors):
    return [s for t in tensors for s in t.stride()[:3]]


def backward_args(q, k, dq, dk, dst, rstd, weights, positions, f, interleaved, workspace, d_weight=(None, None), dst_strides=None):
    batch, length, _, head = q.shape
    return packed(_abi.HEAD_NORM_FIELDS, _abi.HEAD_NORM_ARGS, {
        "batch": batch, "length": length, "head_dim": head, "rotary_dim": 2 * len(f), "heads": [q.shape[2], k.shape[2]],
        "dst": dst, "dst_strides": dst_strides or strides(q, k), "src": [q, k], "src_strides": strides(q, k), "weight": weights, "rstd": rstd,
        "positions": positions, "position_strides": positions.stride(), "frequencies": f, "position_dtype": 3,
        "weight_dtype": TYPES[q.dtype], "scale": 1.25, "weight_offset": 0.5, "eps": 1e-6, "interleaved": int(interleaved),
        "d_out": [dq, dk], "d_out_strides": strides(dq, dk), "d_weight": d_weight, "workspace": workspace,
        "workspace_bytes": workspace.numel()})


def heads_case(lm, dtype, interleaved, head, part, length=37):
    g = torch.Generator().manual_seed(head)
    make = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    q, k, dq, dk = make(2, length, 6, head), make(2, length, 2, head), make(2, length, 6, head), make(2, length, 2, head)
    w = [make(head), make(head)]
    positions = torch.randint(0, 4096, (2, length), generator=g, dtype=torch.int32).cuda()
    f = lm.rotary_frequencies(part)[0]
    how = dict(q_weight=w[0], k_weight=w[1], weight_offset=0.5, scale=1.25, interleaved=interleaved)
    o = lm.head_norm_rotary(q, k, positions, f, **how)
    return q, k, dq, dk, w, positions, f, o, how


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head,part", [(128, 128), (80, 32), (66, 50), (3, 2)])
def test_head_norm_gradients_in_place(lm, dtype, interleaved, head, part):
    """Over the gradients that come in and over the inputs, by whole accesses and by single elements."""
    q, k, dq, dk, w, positions, f, o, how = heads_case(lm, dtype, interleaved, head, part)
    want = lm.head_norm_rotary_backward(dq, dk, q, k, positions, f, q_rstd=o.q_rstd, k_rstd=o.k_rstd, **how)
    workspace = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    for over in ("d_out", "src"):
        a, b, c, d = (x.clone() for x in (q, k, dq, dk))
        dst = (c, d) if over == "d_out" else (a, b)
        dw = torch.empty(2, head, device="cuda")
        args = backward_args(a, b, c, d, dst, [o.q_rstd, o.k_rstd], w, positions, f, interleaved, workspace, (dw[0], dw[1]))
        _abi.check(_abi.lib().mtxc_head_norm_rotary_backward(TYPES[dtype], args))
        assert torch.equal(dst[0], want.q) and torch.equal(dst[1], want.k), over
        assert torch.equal(dw[0], want.q_weight) and torch.equal(dw[1], want.k_weight), over


def test_head_norm_outputs_over_other_inputs_are_refused(lm):
    dtype, head = torch.float32, 64
    q, _, dq, _, w, positions, f, _, _ = heads_case(lm, dtype, False, head, 64)
    k, dk = q.clone(), dq.clone()
    a, b, r = torch.empty_like(q), torch.empty_like(q), [torch.ones(q.shape[:3], device="cuda") for _ in range(2)]
    workspace = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    before = [x.clone() for x in (q, k, dq, dk, *r, *w)]
    lib = _abi.lib()

    def backward(dst, d_weight=(None, None)):
        return lib.mtxc_head_norm_rotary_backward(0, backward_args(q, k, dq, dk, dst, r, w, positions, f, False, workspace, d_weight))

    for dst in ((dk, b), (a, dq), (k, b), (a, q), (dk, dq), (r[0], b), (a, w[1])):
        assert backward(dst) == _abi.ERR_INVALID_ARGUMENT
    for d_weight in ((r[0], None), (None, r[1]), (w[1], None), (q, None), (None, dk)):
        assert backward((a, b), d_weight) == _abi.ERR_INVALID_ARGUMENT
    out = lm.head_norm_rotary(q, k, positions, f)
    for rstd in ((q, None), (None, w[0]), (w[1], None)):
        args = backward_args(q, k, dq, dk, (a, b), rstd, w, positions, f, False, workspace)
        assert lib.mtxc_head_norm_rotary(0, args) == _abi.ERR_INVALID_ARGUMENT
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip((q, k, dq, dk, *r, *w), before))
    assert backward((a, b)) == 0 and torch.isfinite(out.q).all()


def test_outputs_over_their_input_in_another_order_are_refused(lm):
    """Axes exchanged: elements would be written before they are read.  Strides of axes of one element do not count."""
    q = torch.randn(4, 4, 64, device="cuda")
    turned, before = q.transpose(0, 1), q.clone()
    starts, positions = torch.tensor([0, 4], dtype=torch.int32).cuda(), torch.arange(4, dtype=torch.int32).cuda()
    f = lm.rotary_frequencies(64)[0]
    cache, table = lm.kv_cache(1, 16, 2, 64, torch.float32), torch.zeros(4, 1, dtype=torch.int32).cuda()
    k = torch.randn(4, 2, 64, device="cuda")
    w, r = [None, None], [torch.ones(1, 4, 4, device="cuda"), torch.ones(1, 4, 2, device="cuda")]
    for call in (lambda: lm.head_norm_rotary(q, None, positions, f, out=(turned, None)),
                 lambda: lm.head_norm_rotary(k, q, positions, f, out=(torch.empty_like(k), turned)),
                 lambda: lm.decode_attention(q, cache, table, positions, out=turned),
                 lambda: lm.prompt_attention(q, k, k, starts, out=turned)):
        with pytest.raises(MtxcError) as e:
            call()
        assert e.value.code == _abi.ERR_INVALID_ARGUMENT
    dq, dk = torch.randn(1, 4, 4, 64, device="cuda"), torch.randn(1, 4, 2, 64, device="cuda")
    before_dq, workspace = dq.clone(), torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    for q4 in (q[None], dq):  # over src, over d_out
        args = {"q": q[None], "k": k[None], "dq": dq, "dk": dk, "rstd": r, "weights": w, "positions": positions[None], "f": f,
                "interleaved": False, "workspace": workspace}
        over = torch.as_strided(q4, (1, 4, 4, 64), (1024, 64, 256, 1))
        packed_args = backward_args(dst=(over, torch.empty_like(dk)), dst_strides=strides(over, dk), **args)
        assert _abi.lib().mtxc_head_norm_rotary_backward(0, packed_args) == _abi.ERR_INVALID_ARGUMENT
    torch.cuda.synchronize()
    assert torch.equal(q, before) and torch.equal(dq, before_dq)
    one = torch.randn(1, 4, 64, device="cuda")
    want = lm.prompt_attention(one, one, one, starts[:2] // 4)
    assert torch.equal(lm.prompt_attention(one.clone(), one, one, starts // 4, out=None), want)
    again = one.clone()
    odd = torch.as_strided(again, (1, 4, 64), (7, 64, 1))
    assert torch.equal(lm.prompt_attention(again, one, one, starts // 4, out=odd), want)


def test_one_tensor_for_both_exponents(lm):
    """Read by every call, written by none: keys and values have different scales."""
    e4m3 = torch.float8_e4m3fn
    cache = lm.kv_cache(2, 4, 2, 64, e4m3)
    shared = lm.KVCache(cache.keys, cache.values, cache.key_exponents, cache.key_exponents)
    k, slots = torch.randn(8, 2, 64, device="cuda"), torch.arange(8).cuda()
    with pytest.raises(MtxcError) as e:
        lm.cache_write(shared, k, k * 100, slots)
    assert e.value.code == _abi.ERR_INVALID_ARGUMENT
    torch.cuda.synchronize()
    assert not cache.keys.view(torch.uint8).any() and not cache.key_exponents.any()
    lm.cache_write(cache, k, k.flip(0), slots)
    cache.key_exponents.fill_(-7)
    cache.value_exponents.fill_(-7)
    for got, want in zip(lm.cache_read(shared, slots), lm.cache_read(cache, slots)):
        assert torch.equal(got, want)
    table, n = torch.tensor([[0, 1]], dtype=torch.int32).cuda(), torch.tensor([7], dtype=torch.int32).cuda()
    q = torch.randn(1, 4, 64, device="cuda").half()
    assert torch.equal(lm.decode_attention(q, shared, table, n), lm.decode_attention(q, cache, table, n))


def test_a_workspace_off_its_alignment_is_refused(lm):
    q, k, dq, dk, w, positions, f, o, _ = heads_case(lm, torch.float32, False, 64, 64)
    dst, dw = (torch.full_like(q, 7.0), torch.full_like(k, 7.0)), torch.empty(2, 64, device="cuda")
    workspace = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    cache, table = lm.kv_cache(1, 16, 1, 64, torch.float32), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    x, n = torch.ones(1, 2, 64, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(x, 7.0)
    lib = _abi.lib()
    for off, status in ((1, _abi.ERR_INVALID_ARGUMENT), (4, _abi.ERR_INVALID_ARGUMENT), (128, _abi.ERR_INVALID_ARGUMENT), (0, 0)):
        args = backward_args(q, k, dq, dk, dst, [o.q_rstd, o.k_rstd], w, positions, f, False, workspace[off:], (dw[0], dw[1]))
        assert lib.mtxc_head_norm_rotary_backward(0, args) == status
        args = packed(_abi.DECODE_ATTENTION_FIELDS, _abi.DECODE_ATTENTION_ARGS, {
            "cache.pages": 1, "cache.page_size": 16, "cache.heads": 1, "cache.head_dim": 64, "cache.data": cache[:2],
            "cache.strides": strides(*cache[:2]), "batch": 1, "max_pages": 1, "heads": 2, "scale": 0.125, "q": x,
            "q_strides": x.stride()[:2], "out": out, "out_strides": out.stride()[:2], "page_table": table, "page_table_stride": 1,
            "lengths": n, "workspace": workspace[off:], "workspace_bytes": workspace.numel() - off})
        assert lib.mtxc_decode_attention(0, args) == status
        torch.cuda.synchronize()
        assert (out == 7).all() == bool(status) and (dst[0] == 7).all() == bool(status)
    assert not out.any()
