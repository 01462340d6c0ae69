"""The attention operators' argument structs and refusals; on the CPU what needs no device, and on the GPU calls that are
refused before anything runs."""
import ctypes as C
import struct
import subprocess
import threading

import pytest
import torch

from matrix_b200 import MtxcError, _abi, lm
from tests.conftest import REPO
from tests.test_lm import Claimed

STRUCTS = {"mtxc_head_norm_args": _abi.HEAD_NORM_FIELDS, "mtxc_kv_cache": _abi.KV_CACHE_FIELDS,
           "mtxc_cache_rows_args": _abi.CACHE_ROWS_FIELDS, "mtxc_decode_attention_args": _abi.DECODE_ATTENTION_FIELDS,
           "mtxc_prompt_attention_args": _abi.PROMPT_ATTENTION_FIELDS}
CALLS = ("mtxc_head_norm_rotary", "mtxc_head_norm_rotary_backward", "mtxc_cache_write", "mtxc_cache_read", "mtxc_decode_attention",
         "mtxc_prompt_attention")


def test_argument_layouts_match_the_header(tmp_path):
    lines = []
    for name, fields in STRUCTS.items():
        lines += [f'printf("%zu\\n", sizeof({name}));']
        lines += [f'printf("%zu\\n", offsetof({name}, {f.split(":")[0]}));' for f in fields]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mtxc.h"\nint main(void) {' + "".join(lines) +
                   f'printf("%d\\n", MTXC_FLOAT8_E4M3 == {_abi.FLOAT8_E4M3}); return 0; }}')
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    got = []
    for fields in STRUCTS.values():
        types = [f.split(":")[1] for f in fields]
        got.append(struct.calcsize("@" + "".join(types) + "0P"))
        got += [struct.calcsize("@" + "".join(types[:i]) + "0" + t[-1]) for i, t in enumerate(types)]
    assert [int(x) for x in out] == got + [1]


def test_calls_before_init_fail_cleanly():
    """On a thread that is bound to no device."""
    lib, zeros, size = _abi.lib(), b"\0" * 512, C.c_size_t()
    caught = []

    def work():
        caught.extend(getattr(lib, name)(0, zeros) for name in CALLS)
        caught.append(lib.mtxc_decode_attention_workspace(0, zeros, C.byref(size)))
        caught.append(lib.mtxc_head_norm_rotary_backward_workspace(0, zeros, C.byref(size)))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert caught == [_abi.ERR_NOT_INITIALIZED] * 8
    recording = C.c_int(7)
    assert lib.mtxc_graph_recording(C.byref(recording)) == 0 and recording.value == 0
    assert lib.mtxc_graph_recording(None) == _abi.ERR_INVALID_ARGUMENT


def calls_on(make):
    """Each operator once, over tensors that make(*shape, dtype=...) gives."""
    q, pos = make(4, 2, 8), make(4, dtype=torch.int32)
    f, starts = make(4, dtype=torch.float64), make(2, dtype=torch.int32)
    rstd, table = make(4, 2), make(4, 1, dtype=torch.int32)
    cache = lm.KVCache(make(3, 2, 2, 8), make(3, 2, 2, 8))
    return [lambda: lm.head_norm_rotary(q, None, pos, f), lambda: lm.head_norm_rotary_backward(q, None, q, None, pos, f, q_rstd=rstd),
            lambda: lm.cache_write(cache, q, q, pos), lambda: lm.cache_read(cache, pos),
            lambda: lm.decode_attention(q, cache, table, pos), lambda: lm.prompt_attention(q, q, q, starts)]


def test_host_tensors_are_refused():
    for call in calls_on(torch.zeros):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def claimed(device):
    return lambda *shape, dtype=torch.float32: Claimed(device, *shape, dtype=dtype)


def test_a_thread_without_a_device_is_refused():
    caught = []

    def work():
        for call in calls_on(claimed("cuda:0")):
            try:
                caught.append(call())
            except MtxcError as e:
                caught.append(e.code)
            except Exception as e:  # noqa: BLE001
                caught.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert caught == [_abi.ERR_NOT_INITIALIZED] * 6


def test_kv_cache_shapes():
    c = lm.kv_cache(3, 4, 2, 8, torch.float16, device="cpu")
    assert c.keys.shape == (3, 4, 2, 8) and c.keys.stride() == (64, 8, 32, 1) and c.key_exponents is None
    assert not c.keys.any() and c.values.data_ptr() != c.keys.data_ptr()
    c = lm.kv_cache(3, 4, 2, 8, torch.float8_e4m3fn, device="cpu")
    assert c.values.dtype == torch.float8_e4m3fn and c.value_exponents.shape == (3, 4, 2)
    assert c.value_exponents.dtype == torch.int8 and c.value_exponents.stride() == (8, 1, 4)


def test_attention_takes_tensors():
    for call in (lambda: lm.cache_read(lm.KVCache(None, None), None, dtype=torch.float32),
                 lambda: lm.decode_attention(None, lm.KVCache(None, None), None, None), lambda: lm.prompt_attention(1, 2, 3, 4),
                 lambda: lm.head_norm_rotary(1, None, 2, 3)):
        with pytest.raises(TypeError, match="expected a tensor"):
            call()


@pytest.mark.gpu
def test_tensors_of_another_device_are_refused(gpu):
    for call in calls_on(claimed("cuda:1")):
        with pytest.raises(ValueError, match="cuda:0, the device that the thread is bound to"):
            call()


def cuda(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


@pytest.mark.gpu
def test_head_norm_refusals(gpu):
    q, k, pos, f = cuda(2, 4, 3, 8), cuda(2, 4, 1, 8), cuda(4, dtype=torch.int32), cuda(4, dtype=torch.float64)
    w, r, other = cuda(8), cuda(2, 4, 3), cuda(2, 4, 3, 8)
    bad = [
        lambda: lm.head_norm_rotary(cuda(4, 8), None, pos, f),
        lambda: lm.head_norm_rotary(q, cuda(2, 4, 1, 6), pos, f),
        lambda: lm.head_norm_rotary(q, k.half(), pos, f),
        lambda: lm.head_norm_rotary(q, cuda(2, 5, 1, 8), pos, f),
        lambda: lm.head_norm_rotary(q, k, pos.float(), f),
        lambda: lm.head_norm_rotary(q, k, pos[:3], f),
        lambda: lm.head_norm_rotary(q, k, cuda(3, 4, dtype=torch.int32), f),
        lambda: lm.head_norm_rotary(q, k, pos, f.float()),
        lambda: lm.head_norm_rotary(q, k, pos, cuda(8, dtype=torch.float64)[::2]),
        lambda: lm.head_norm_rotary(q, k, pos, f, q_weight=cuda(7)),
        lambda: lm.head_norm_rotary(q, k, pos, f, q_weight=cuda(16)[::2]),
        lambda: lm.head_norm_rotary(q, k, pos, f, q_weight=w, k_weight=w.half()),
        lambda: lm.head_norm_rotary(q, None, pos, f, k_weight=w),
        lambda: lm.head_norm_rotary(q.transpose(2, 3), None, pos, cuda(1, dtype=torch.float64)),
        lambda: lm.head_norm_rotary(q, k, pos, f, out=(cuda(2, 4, 3, 7), None)),
        lambda: lm.head_norm_rotary(q, k, pos, f, out=(cuda(2, 4, 1, 8).expand(2, 4, 3, 8), None)),
        lambda: lm.head_norm_rotary_backward(cuda(2, 4, 3, 6), None, q, None, pos, f, q_rstd=r),
        lambda: lm.head_norm_rotary_backward(q.half(), None, q, None, pos, f, q_rstd=r),
        lambda: lm.head_norm_rotary_backward(q, None, q, k, pos, f, q_rstd=r),
        lambda: lm.head_norm_rotary_backward(q, k, q, k, pos, f, q_rstd=r),
        lambda: lm.head_norm_rotary_backward(q, None, q, None, pos, f, q_rstd=r[:1]),
        lambda: lm.head_norm_rotary_backward(q, None, q, None, pos, f, q_rstd=r.double()),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call, code in [(lambda: lm.head_norm_rotary(q, k, pos, cuda(5, dtype=torch.float64)), _abi.ERR_INVALID_ARGUMENT),
                       (lambda: lm.head_norm_rotary(q.double(), None, pos, f), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.head_norm_rotary(q, k, pos, f, q_weight=w.int()), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.head_norm_rotary(q, q, pos, f, out=(q, q)), _abi.ERR_INVALID_ARGUMENT),
                       (lambda: lm.head_norm_rotary(q, other, pos, f, out=(other, q)), _abi.ERR_INVALID_ARGUMENT),
                       (lambda: lm.head_norm_rotary(cuda(1, 1, 1, 1025), None, pos[:1], f), _abi.ERR_SHAPE)]:
        with pytest.raises(MtxcError) as e:
            call()
        assert e.value.code == code


@pytest.mark.gpu
def test_cache_refusals(gpu):
    cache, small = lm.kv_cache(3, 4, 2, 8, torch.float32), lm.kv_cache(3, 4, 2, 8, torch.float8_e4m3fn)
    one = lm.KVCache(*(cuda(1, 4, 2, 8) for _ in range(2)))
    k, slots = cuda(5, 2, 8), cuda(5, dtype=torch.int32)
    bad = [
        lambda: lm.cache_write(cache, k, k, slots.float()),
        lambda: lm.cache_write(cache, k, k, slots[:4]),
        lambda: lm.cache_write(cache, k, k, slots[None]),
        lambda: lm.cache_write(cache, k[:, :1], k, slots),
        lambda: lm.cache_write(cache, k, k[:, :, :7], slots),
        lambda: lm.cache_write(cache, k, k.half(), slots),
        lambda: lm.cache_write(cache, cuda(5, 8, 2).transpose(1, 2), k, slots),
        lambda: lm.cache_write(lm.KVCache(cache.keys, cache.values[:2]), k, k, slots),
        lambda: lm.cache_write(lm.KVCache(cache.keys, cache.values.half()), k, k, slots),
        lambda: lm.cache_write(lm.KVCache(cache.keys[0], cache.values[0]), k, k, slots),
        lambda: lm.cache_write(lm.KVCache(*small[:2]), k, k, slots),
        lambda: lm.cache_write(lm.KVCache(*cache[:2], *small[2:]), k, k, slots),
        lambda: lm.cache_write(lm.KVCache(*small[:3], small.value_exponents.int()), k, k, slots),
        lambda: lm.cache_write(lm.KVCache(*small[:3], small.value_exponents[:2]), k, k, slots),
        lambda: lm.cache_write(lm.KVCache(cache.keys[:1].expand(3, 4, 2, 8), cache.values), k, k, slots),
        lambda: lm.cache_write(lm.KVCache(*small[:3], small.value_exponents[:1].expand(3, 4, 2)), k, k, slots),
        lambda: lm.cache_read(small, slots, dtype=torch.float64),
        lambda: lm.cache_read(cache, slots, out=(k, cuda(5, 2, 7))),
        lambda: lm.cache_read(cache, slots, out=(cuda(5, 1, 8).expand(5, 2, 8), k)),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call, code in [(lambda: lm.cache_write(cache, k.half(), k.half(), slots), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.cache_write(small, k.int(), k.int(), slots), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.cache_write(lm.KVCache(cache.keys, cache.keys), k, k, slots), _abi.ERR_INVALID_ARGUMENT),
                       (lambda: lm.cache_read(cache, slots, dtype=torch.float16), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.cache_read(cache, slots, out=(k, k)), _abi.ERR_INVALID_ARGUMENT),
                       (lambda: lm.cache_read(one, slots[:4], out=(one.keys[0], k[:4])), _abi.ERR_INVALID_ARGUMENT),
                       (lambda: lm.cache_write(one, one.keys[0], k[:4], slots[:4]), _abi.ERR_INVALID_ARGUMENT),
                       (lambda: lm.cache_write(lm.kv_cache(1, 1, 1, 1025, torch.float32), cuda(5, 1, 1025), cuda(5, 1, 1025), slots),
                        _abi.ERR_SHAPE)]:
        with pytest.raises(MtxcError) as e:
            call()
        assert e.value.code == code
    with pytest.raises(TypeError):
        lm.cache_read(cache, slots, dtype="float32")


@pytest.mark.gpu
def test_decode_refusals(gpu):
    cache, q = lm.kv_cache(3, 4, 2, 8, torch.float32), cuda(2, 4, 8)
    table, n = cuda(2, 3, dtype=torch.int32), cuda(2, dtype=torch.int32)
    one = lm.KVCache(*(cuda(1, 4, 2, 8) for _ in range(2)))
    bad = [
        lambda: lm.decode_attention(q[0], cache, table, n),
        lambda: lm.decode_attention(cuda(2, 4, 6), cache, table, n),
        lambda: lm.decode_attention(cuda(2, 8, 4).transpose(1, 2), lm.kv_cache(3, 4, 2, 8, torch.float32), table, n),
        lambda: lm.decode_attention(q, cache, table.long(), n),
        lambda: lm.decode_attention(q, cache, table[:1], n),
        lambda: lm.decode_attention(q, cache, cuda(3, 2, dtype=torch.int32).T, n),
        lambda: lm.decode_attention(q, cache, table, n.long()),
        lambda: lm.decode_attention(q, cache, table, n[:1]),
        lambda: lm.decode_attention(q, cache, table, cuda(4, dtype=torch.int32)[::2]),
        lambda: lm.decode_attention(q, cache, table, n, out=cuda(2, 4, 7)),
        lambda: lm.decode_attention(q, cache, table, n, out=cuda(2, 1, 8).expand(2, 4, 8)),
        lambda: lm.decode_attention(q, lm.KVCache(cache.keys, cache.values[:, :, :1]), table, n),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call, code in [(lambda: lm.decode_attention(q.half(), cache, table, n), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.decode_attention(q.double(), cache, table, n), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.decode_attention(cuda(2, 3, 8), cache, table, n), _abi.ERR_SHAPE),
                       (lambda: lm.decode_attention(cuda(1, 2, 8), one, table[:1], n[:1], out=one.values[0, :1]), _abi.ERR_INVALID_ARGUMENT),
                       (lambda: lm.decode_attention(cuda(2, 2, 257), lm.kv_cache(1, 1, 1, 257, torch.float32), table, n), _abi.ERR_SHAPE),
                       (lambda: lm.decode_attention(q, lm.kv_cache(1, 0, 2, 8, torch.float32), table, n), _abi.ERR_SHAPE)]:
        with pytest.raises(MtxcError) as e:
            call()
        assert e.value.code == code


@pytest.mark.gpu
def test_prompt_refusals(gpu):
    q, k, starts, other = cuda(6, 4, 8), cuda(6, 2, 8), cuda(3, dtype=torch.int32), cuda(6, 4, 8)
    bad = [
        lambda: lm.prompt_attention(q[0], k, k, starts),
        lambda: lm.prompt_attention(q, cuda(6, 2, 6), k, starts),
        lambda: lm.prompt_attention(q, k.half(), k.half(), starts),
        lambda: lm.prompt_attention(q, k, k[:5], starts),
        lambda: lm.prompt_attention(q, k, k.half(), starts),
        lambda: lm.prompt_attention(q, k[:5], k[:5], starts),
        lambda: lm.prompt_attention(q, k, k, starts.long()),
        lambda: lm.prompt_attention(q, k, k, starts[:0]),
        lambda: lm.prompt_attention(q, k, k, starts[0]),
        lambda: lm.prompt_attention(q, k, k, starts, k_starts=starts[:2]),
        lambda: lm.prompt_attention(q, k, k, cuda(6, dtype=torch.int32)[::2]),
        lambda: lm.prompt_attention(cuda(6, 8, 4).transpose(1, 2), k, k, starts),
        lambda: lm.prompt_attention(q, k, cuda(6, 8, 2).transpose(1, 2), starts),
        lambda: lm.prompt_attention(q, k, k, starts, out=cuda(6, 4, 7)),
        lambda: lm.prompt_attention(q, k, k, starts, out=cuda(1, 4, 8).expand(6, 4, 8)),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call, code in [(lambda: lm.prompt_attention(q.double(), k.double(), k.double(), starts), _abi.ERR_UNSUPPORTED_DTYPE),
                       (lambda: lm.prompt_attention(cuda(6, 3, 8), k, k, starts), _abi.ERR_SHAPE),
                       (lambda: lm.prompt_attention(q, q, other, starts, out=other), _abi.ERR_INVALID_ARGUMENT),
                       (lambda: lm.prompt_attention(cuda(6, 2, 257), cuda(6, 2, 257), cuda(6, 2, 257), starts), _abi.ERR_SHAPE)]:
        with pytest.raises(MtxcError) as e:
            call()
        assert e.value.code == code
