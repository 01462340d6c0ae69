"""Row operators of a language model on device tensors: the norms around a block with its gate, dropout and
residual, dropout by itself, rotary positions, and the rules on logits before a token is chosen.

These functions hand a call's tensors to the C ABI (include/mtxc.h, which states the formulas) through the module
that matrix_b200/binding compiles against torch; PyTorch only provides device memory and streams, and there is no
autograd: an operator's backward pass is a function of its own.  ``backend.init`` binds the thread first.  Kernels
run on the thread's stream (``backend.set_stream``), and the outputs made here come from that stream's memory;
where it is not torch's current stream, ordering the two is the caller's, as for any two streams.  A tensor given as
an output counts as changed in place.

Inputs are float32, float16 or bfloat16 tensors on the thread's device whose last axis has unit stride; the other axes
of a row operator's inputs have to fold into one axis of rows (a constant stride from row to row).
"""
from __future__ import annotations

import ctypes
import importlib.util
from typing import NamedTuple

import torch

from . import _abi
from ._abi import check, lib

__all__ = ["BlockNorm", "BlockNormGradients", "block_norm", "block_norm_backward", "dropout", "logits_rules", "rotary",
           "rotary_frequencies"]


def _load():
    path = _abi.LIB_PATH.with_name("_lm.so")
    if not path.exists():
        raise ImportError(f"{path} not found: build it with `python -m matrix_b200.build`")
    lib()  # the library that the module calls, from the same place
    spec = importlib.util.spec_from_file_location("matrix_b200._lm", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    if module.torch_version != torch.__version__:
        raise ImportError(f"{path} was compiled against torch {module.torch_version}, not the installed {torch.__version__}: "
                          "build it again with `python -m matrix_b200.build`")
    return module


_lm = _load()


def _done(r):
    """What the module returned: outputs, or the C ABI's status."""
    if r.__class__ is int:
        check(r)
    return r


def dropout(x: torch.Tensor, p: float, seed: int, offset: int, *, device_offset: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """x with elements dropped with probability p and the others divided by 1 - p (both to 16 bits), by the
    counter-based generator of mtxc_dropout.  With the same seed and offset it is its own backward pass
    (gradients for x); every call of a step needs an offset of its own.  device_offset: one 64-bit integer on
    the device, added to offset when the kernel runs.  out may be x."""
    return _done(_lm.dropout(x, p, seed, offset, device_offset, out))[0]


class BlockNorm(NamedTuple):
    """What block_norm returns; None where the call has no such output."""

    residual: torch.Tensor
    normed: torch.Tensor | None
    post_rstd: torch.Tensor | None
    next_rstd: torch.Tensor | None


class BlockNormGradients(NamedTuple):
    """Gradients of block_norm's inputs; None where the call has no such input."""

    residual: torch.Tensor
    branch: torch.Tensor | None
    post_weight: torch.Tensor | None
    gate: torch.Tensor | None
    next_weight: torch.Tensor | None


def block_norm(residual: torch.Tensor, branch: torch.Tensor | None = None, *, post_weight: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, next_weight: torch.Tensor | None = None, residual_scale: float = 1.0,
               branch_scale: float = 1.0, weight_offset: float = 0.0, eps: float = 1e-6, dropout: float = 0.0,
               seed: int = 0, offset: int = 0, device_offset: torch.Tensor | None = None, save_rstd: bool = True,
               out: torch.Tensor | None = None, normed_out: torch.Tensor | None = None) -> BlockNorm:
    """The norms after and before a block in one pass (mtxc_block_norm):

        residual' = residual_scale * residual + branch_scale * gate * dropout(rms_norm(branch) * post_weight)
        normed    = rms_norm(residual') * next_weight

    Without post_weight the branch is not normed, without next_weight there is no normed, without a branch
    this is the norm in front of the first block (and the residual itself is returned, unless it is scaled).
    The gate is one row of the width (a gate per channel), or has the residual's leading axes with the last
    ones of extent 1 ([batch, 1, width]: one per sequence; the full shape: one per token).  Weights are
    multiplied as weight_offset + weight.  save_rstd: keep the norms' reciprocal deviations (one float per
    row) for block_norm_backward.  out and normed_out may be the residual and the branch."""
    return BlockNorm._make(_done(_lm.block_norm(residual, branch, post_weight, gate, next_weight, residual_scale,
                                                branch_scale, weight_offset, eps, dropout, seed, offset, device_offset,
                                                save_rstd, out, normed_out)))


def block_norm_backward(d_residual: torch.Tensor | None, d_normed: torch.Tensor | None, residual: torch.Tensor,
                        branch: torch.Tensor | None = None, *, post_rstd: torch.Tensor | None = None,
                        next_rstd: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                        gate: torch.Tensor | None = None, next_weight: torch.Tensor | None = None,
                        residual_scale: float = 1.0, branch_scale: float = 1.0, weight_offset: float = 0.0,
                        dropout: float = 0.0, seed: int = 0, offset: int = 0,
                        device_offset: torch.Tensor | None = None, parameters: bool = True) -> BlockNormGradients:
    """The gradients of block_norm's inputs (mtxc_block_norm_backward), given those of its outputs (d_residual
    None: zero; d_normed None: there is no next_weight), the residual that it returned, its branch and the
    saved rstds, with the forward call's other arguments.  The weights' gradients are float32; the gate's has
    the gate's shape and dtype.  parameters=False: none of the three is wanted."""
    return BlockNormGradients._make(_done(_lm.block_norm_backward(
        d_residual, d_normed, residual, branch, post_rstd, next_rstd, post_weight, gate, next_weight, residual_scale,
        branch_scale, weight_offset, dropout, seed, offset, device_offset, parameters)))


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                       original_length: float = 0.0, fast_turns: float = 32.0, slow_turns: float = 1.0,
                       device="cuda") -> tuple[torch.Tensor, float]:
    """The frequencies (float64, rotary_dim / 2 of them, on the device) and the scale that `rotary` takes, for
    a context `factor` times as long as the one trained on: scaling "none", "linear", "base" or "by_parts"
    (mtxc_rotary_frequencies states them)."""
    if not 0 <= rotary_dim < 1 << 31:  # the C ABI takes 32 bits, and fills as many values as they say
        raise ValueError("rotary_dim: expected 0 .. 2^31 - 1")
    values = (ctypes.c_double * max(1, rotary_dim // 2))()
    scale = ctypes.c_double()
    if scaling not in _abi.ROTARY_SCALINGS:
        raise ValueError(f"scaling: expected one of {sorted(_abi.ROTARY_SCALINGS)}")
    check(lib().mtxc_rotary_frequencies(_abi.ROTARY_SCALINGS[scaling], rotary_dim, base, factor, original_length,
                                        fast_turns, slow_turns, values, ctypes.byref(scale)))
    return torch.tensor(values[:rotary_dim // 2], dtype=torch.float64, device=device), scale.value


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, frequencies: torch.Tensor, *,
           scale: float = 1.0, interleaved: bool = False, inverse: bool = False,
           out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Queries and keys turned by their positions (mtxc_rotary), in one launch: q and k are [batch, length,
    heads, head_dim] or [length, heads, head_dim] with any strides (heads may be stored before tokens) but unit
    stride within a head; k may have fewer heads, or be None.  positions: int32 or int64, [batch, length] or
    [length].  frequencies and scale: as rotary_frequencies gives them; the first 2 * len(frequencies) elements
    of a head are turned, in pairs (j, j + half) or, interleaved, (2j, 2j + 1), and the others passed on.
    inverse=True is the backward pass.  out=(q, k) writes in place."""
    q_out, k_out = out if out is not None else (None, None)
    return _done(_lm.rotary(q, k, positions, frequencies, scale, interleaved, inverse, q_out, k_out))


def logits_rules(logits: torch.Tensor, *, tokens: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                 prompt_lengths: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                 frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                 bias_tokens: torch.Tensor | None = None, bias_values: torch.Tensor | None = None,
                 mask: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Logits [rows, vocab] after the rules that precede the choice of a token (mtxc_logits_rules), each of
    which may be absent: penalties for the tokens of a row (tokens int32 [rows, n], of which the first
    lengths[row] count and the first prompt_lengths[row] are the prompt's; repetition, frequency and presence
    float32 [rows]), biases (bias_tokens int32, bias_values float32, [rows, m] or [m]; the last entry for a
    token counts) and a mask of allowed tokens (int32 words [rows, ceil(vocab / 32)] or [ceil(vocab / 32)], bit
    v % 32 of word v / 32).  Lists may hold padding outside the vocabulary.  out may be logits."""
    return _done(_lm.logits_rules(logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias_tokens,
                                  bias_values, mask, out))[0]
