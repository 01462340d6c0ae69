"""Waits inside kernels: bounded, and reported (mtxc_waits_gave_up)."""
import ctypes as C
import subprocess
import threading

import pytest
import torch

from matrix_b200 import _abi, build
from tests.conftest import REPO


def test_query_refusals():
    lib, caught = _abi.lib(), []
    assert lib.mtxc_waits_gave_up(None) == _abi.ERR_INVALID_ARGUMENT
    t = threading.Thread(target=lambda: caught.append(lib.mtxc_waits_gave_up(C.byref(C.c_int()))))
    t.start()
    t.join()
    assert caught == [_abi.ERR_NOT_INITIALIZED]


@pytest.mark.gpu
@pytest.mark.parametrize("head", [64, 128, 256])
def test_no_wait_gave_up(gpu, head):
    from matrix_b200 import lm

    x = torch.randn(300, 2, head, device="cuda").bfloat16()
    lm.prompt_attention(x, x, x, torch.tensor([0, 100, 300], dtype=torch.int32).cuda())
    assert lm.waits_gave_up() is False


@pytest.mark.gpu
def test_a_wait_runs_out(gpu, tmp_path):
    """About four seconds, and a flag; no fault, and nothing that is left behind."""
    exe = tmp_path / "test_waits"
    subprocess.run([build.nvcc(), *build.ARCH, *build.NVCC_FLAGS, str(REPO / "tests" / "cpp" / "test_waits.cu"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout + run.stderr
    first, failed, second, third, fourth, first_cycles, second_cycles = map(int, run.stdout.split())
    assert (first, failed, second, third, fourth) == (0, 1, 0, 1, 1)
    assert 1e9 < first_cycles < 6e10 and second_cycles < 1e6
