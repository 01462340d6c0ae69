"""The build of the module over torch tensors: which torch it is for, and what happens without one."""
import sys

import pytest
import torch

from matrix_b200 import build, lm


@pytest.fixture
def elsewhere(monkeypatch, tmp_path):
    """The module and its record in an empty folder, and a compiler that only writes down its commands."""
    monkeypatch.setattr(build, "BINDING_LIB", tmp_path / "_lm.so")
    monkeypatch.setattr(build, "BINDING_TORCH", tmp_path / "_lm.torch")
    commands = []

    def run(cmd, verbose=False):
        commands.append(cmd)
        (tmp_path / "_lm.so").touch()
        return ""

    monkeypatch.setattr(build, "_run", run)
    return commands


def test_without_torch_the_module_is_left_out(elsewhere, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # import torch raises ImportError
    assert build.build_binding([]) is None
    assert not elsewhere and not build.BINDING_LIB.exists()
    assert "_lm.so left out" in capsys.readouterr().err


def test_with_a_torch_without_cuda_the_module_is_left_out(elsewhere, monkeypatch, capsys):
    monkeypatch.setattr(torch.version, "cuda", None)
    assert build.build_binding([]) is None
    assert not elsewhere and "without CUDA" in capsys.readouterr().err


def test_another_torch_compiles_the_module_again(elsewhere, monkeypatch):
    assert build.build_binding([]) == build.BINDING_LIB and len(elsewhere) == 1
    build.build_binding([])
    assert len(elsewhere) == 1  # up to date
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build_binding([])
    assert len(elsewhere) == 2 and '-DMTX_TORCH_VERSION="0.0.1"' in elsewhere[1]


def test_a_module_for_another_torch_is_not_loaded(monkeypatch):
    assert lm._lm.torch_version == torch.__version__
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    with pytest.raises(ImportError, match="0.0.1"):
        lm._load()
