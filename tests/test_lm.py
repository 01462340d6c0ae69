"""The language-model row operators without a GPU: the generator's known answers, the frequencies, the layout
of the argument structs, and the refusals that need no device."""
import ctypes as C
import math
import subprocess
import threading

import numpy as np
import pytest
import torch

from matrix_b200 import MtxcError, _abi, lm
from tests import lm_reference as ref
from tests.conftest import REPO


@pytest.mark.parametrize("counter,key,words", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_reference_generator_known_answers(counter, key, words):
    """The published test vectors of Philox4x32-10, for the generator that the kernels are compared with."""
    assert tuple(int(w) for w in ref.philox(counter, key)) == words


STRUCTS = {"mtxc_dropout_state": _abi.DROPOUT_FIELDS, "mtxc_block_norm_args": _abi.BLOCK_NORM_FIELDS,
           "mtxc_block_norm_backward_args": _abi.BLOCK_NORM_BACKWARD_FIELDS, "mtxc_rotary_args": _abi.ROTARY_FIELDS,
           "mtxc_logits_args": _abi.LOGITS_FIELDS}


def test_argument_layouts_match_the_header(tmp_path):
    """Every field that the binding packs lies where the C compiler puts it."""
    lines = []
    for name, fields in STRUCTS.items():
        lines += [f'printf("%zu\\n", sizeof({name}));']
        lines += [f'printf("%zu\\n", offsetof({name}, {f.split(":")[0]}));' for f in fields]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "mtxc.h"\nint main(void) {' + "".join(lines) + "return 0; }")
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    want = [int(v) for v in out]
    import struct

    got = []
    for fields in STRUCTS.values():
        types = [f.split(":")[1] for f in fields]
        got.append(struct.calcsize("@" + "".join(types) + "0P"))
        got += [struct.calcsize("@" + "".join(types[:i]) + "0" + t[-1]) for i, t in enumerate(types)]
    assert got == want


def test_frequencies():
    for dim, base in ((2, 10000.0), (64, 10000.0), (128, 500000.0)):
        f, scale = lm.rotary_frequencies(dim, base, device="cpu")
        want = base ** (-np.arange(0, dim, 2) / dim)
        assert f.dtype == torch.float64 and scale == 1.0
        np.testing.assert_allclose(f.numpy(), want, rtol=1e-14)
        f, _ = lm.rotary_frequencies(dim, base, scaling="linear", factor=4, device="cpu")
        np.testing.assert_allclose(f.numpy(), want / 4, rtol=1e-14)
    f, scale = lm.rotary_frequencies(64, scaling="base", factor=8, device="cpu")
    want = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    assert scale == 1.0 and f[0] == 1.0
    np.testing.assert_allclose(f[-1], want[-1] / 8, rtol=1e-12)  # the slowest is divided by the factor
    f, scale = lm.rotary_frequencies(64, scaling="by_parts", factor=16, original_length=4096, device="cpu")
    turns = 4096 * want / (2 * math.pi)
    assert scale == pytest.approx(0.1 * math.log(16) + 1, rel=1e-15)
    np.testing.assert_allclose(f.numpy()[turns >= 32], want[turns >= 32], rtol=1e-14)
    np.testing.assert_allclose(f.numpy()[turns <= 1], want[turns <= 1] / 16, rtol=1e-14)
    part = (turns > 1) & (turns < 32)
    keep = (turns[part] - 1) / 31
    assert part.any()
    np.testing.assert_allclose(f.numpy()[part], want[part] * (keep + (1 - keep) / 16), rtol=1e-12)
    assert len(lm.rotary_frequencies(0, device="cpu")[0]) == 0


@pytest.mark.parametrize("kwargs", [dict(rotary_dim=7), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, factor=-1.0),
                                    dict(rotary_dim=2, scaling="base", factor=2.0),
                                    dict(rotary_dim=8, scaling="by_parts", factor=2.0),
                                    dict(rotary_dim=8, scaling="by_parts", original_length=10, fast_turns=1, slow_turns=1),
                                    dict(rotary_dim=8, base=float("nan"))])
def test_frequency_refusals(kwargs):
    with pytest.raises(MtxcError) as e:
        lm.rotary_frequencies(**kwargs, device="cpu")
    assert e.value.code == _abi.ERR_INVALID_ARGUMENT
    with pytest.raises(ValueError):
        lm.rotary_frequencies(8, scaling="unknown", device="cpu")


def test_calls_before_init_fail_cleanly():
    lib = _abi.lib()
    zeros = b"\0" * 512
    assert lib.mtxc_dropout(0, None, None, 1, 1, 1, 1, zeros) == _abi.ERR_NOT_INITIALIZED
    for f in (lib.mtxc_block_norm, lib.mtxc_block_norm_backward, lib.mtxc_rotary, lib.mtxc_logits_rules):
        assert f(0, zeros) == _abi.ERR_NOT_INITIALIZED
    one = (C.c_double * 1)()
    assert lib.mtxc_rotary_frequencies(0, 2, 10.0, 1.0, 0.0, 0.0, 0.0, one, None) == _abi.ERR_INVALID_ARGUMENT
    assert lib.mtxc_rotary_frequencies(9, 2, 10.0, 1.0, 0.0, 0.0, 0.0, one, one) == _abi.ERR_INVALID_ARGUMENT


def test_host_tensors_are_refused():
    """A host pointer must not reach a kernel."""
    x = torch.zeros(4, 8)
    f = torch.ones(4, dtype=torch.float64)
    calls = [lambda: lm.dropout(x, 0.5, 0, 0), lambda: lm.block_norm(x, x), lambda: lm.block_norm_backward(x, None, x, x),
             lambda: lm.rotary(x[None], None, torch.zeros(1, dtype=torch.int32), f), lambda: lm.logits_rules(x)]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA"):
            call()


class Claimed(torch.Tensor):
    """A tensor that claims a device and has no memory."""

    @staticmethod
    def __new__(cls, device, *shape, dtype=torch.float32):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device=device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} of a tensor without memory")


def calls_on(device):
    x, q = Claimed(device, 4, 8), Claimed(device, 4, 1, 8)
    f, pos = Claimed(device, 4, dtype=torch.float64), Claimed(device, 4, dtype=torch.int32)
    return [lambda: lm.dropout(x, 0.5, 0, 0), lambda: lm.block_norm(x, x), lambda: lm.block_norm_backward(x, None, x, x),
            lambda: lm.rotary(q, None, pos, f), lambda: lm.logits_rules(x)]


def test_a_thread_without_a_device_is_refused():
    """Before anything is allocated or read: on a thread that is bound to no device."""
    caught = []

    def work():
        device = C.c_int(7)
        caught.append(_abi.lib().mtxc_get_device(C.byref(device)))
        for call in calls_on("cuda:0"):
            try:
                caught.append(call())
            except MtxcError as e:
                caught.append(e.code)
            except Exception as e:
                caught.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert caught == [_abi.ERR_NOT_INITIALIZED] * 6


@pytest.mark.gpu
def test_tensors_of_another_device_are_refused(gpu):
    """Tensors on cuda:1, from a thread bound to cuda:0: their pointers must not reach a kernel, and nothing is
    allocated for them."""
    device = C.c_int(7)
    _abi.check(_abi.lib().mtxc_get_device(C.byref(device)))
    assert device.value == 0
    for call in calls_on("cuda:1"):
        with pytest.raises(ValueError, match="cuda:0, the device that the thread is bound to"):
            call()


@pytest.mark.parametrize("rotary_dim", [-1, -2, -(1 << 32), 1 << 31, (1 << 32) + 4])
def test_frequencies_of_no_dimension_are_refused(rotary_dim):
    """Numbers that 32 bits do not hold: the values would be written past their buffer, or not at all."""
    with pytest.raises(ValueError, match="rotary_dim"):
        lm.rotary_frequencies(rotary_dim, device="cpu")
