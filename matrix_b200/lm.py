"""Row operators of a language model on device tensors: the norms around a block with its gate, dropout and
residual, dropout by itself, rotary positions, and the rules on logits before a token is chosen.

Like ``backend``, these functions compute a call's metadata and hand it to the C ABI (include/mtxc.h, which
states the formulas); PyTorch only provides device memory and streams, and there is no autograd: an
operator's backward pass is a function of its own.  ``backend.init`` binds the thread first.  Kernels run on
the thread's stream (``backend.set_stream``), and the outputs made here come from that stream's memory; where
it is not torch's current stream, ordering the two is the caller's, as for any two streams.

Inputs are float32, float16 or bfloat16 tensors whose last axis has unit stride; the other axes of a row
operator's inputs have to fold into one axis of rows (a constant stride from row to row).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _abi
from ._abi import check, lib
from .backend import dtype_code

__all__ = ["BlockNorm", "BlockNormGradients", "block_norm", "block_norm_backward", "dropout", "logits_rules", "rotary",
           "rotary_frequencies"]


# ------------------------------------------------------------------------------------------
# Arguments
# ------------------------------------------------------------------------------------------
def _on_device(x: torch.Tensor, *others) -> int:
    """The CUDA device that all the tensors (None: absent) are on."""
    dev = x.get_device()
    if dev < 0:
        raise ValueError("expected tensors on a CUDA device")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError("expected all tensors on the same CUDA device")
    return dev


def _own_memory(dev: int) -> bool:
    """Whether torch's current stream is the one that the kernels run on."""
    return (lib().mtxc_get_stream() or 0) == torch._C._cuda_getCurrentRawStream(dev)


def _on_stream(dev: int):
    """Makes the stream that the kernels run on torch's current one, so that new tensors come from its memory."""
    return torch.cuda.stream(torch.cuda.ExternalStream(lib().mtxc_get_stream() or 0, device=dev))


def _new(x: torch.Tensor, shape, dtype: torch.dtype, dev: int) -> torch.Tensor:
    """A contiguous tensor on x's device, from the memory of the stream that the kernels run on."""
    if _own_memory(dev):
        return x.new_empty(shape, dtype=dtype)
    with _on_stream(dev):
        return x.new_empty(shape, dtype=dtype)


def _new_like(x: torch.Tensor, dev: int) -> torch.Tensor:
    """The same with x's shape and dtype."""
    if x.is_contiguous():
        if _own_memory(dev):
            return torch.empty_like(x)
        with _on_stream(dev):
            return torch.empty_like(x)
    return _new(x, x.shape, x.dtype, dev)


def _row_stride(t: torch.Tensor, what: str, written: bool = False) -> int:
    """The stride from row to row of a tensor whose leading axes fold into one."""
    shape = t.shape
    width = shape[-1]
    if t.is_contiguous():
        return width
    strides = t.stride()
    n = len(shape)
    if width > 1 and strides[-1] != 1:
        raise ValueError(f"{what}: the last axis needs unit stride")
    stride, span = width, 0  # span: the extent so far times its stride, which the next axis out must continue
    for i in range(n - 2, -1, -1):
        if shape[i] == 1:
            continue
        if span == 0:
            stride = strides[i]
            span = stride * shape[i]
        elif strides[i] == span:
            span *= shape[i]
        else:
            raise ValueError(f"{what}: its leading axes do not fold into rows at a constant stride")
        if written and stride < width:
            raise ValueError(f"{what}: its rows overlap")
    return stride


def _like(x: torch.Tensor, out: torch.Tensor | None, what: str, dev: int) -> torch.Tensor:
    if out is None:
        return _new_like(x, dev)
    if out.shape != x.shape or out.dtype != x.dtype or out.get_device() != dev:
        raise ValueError(f"{what}: expected a tensor of the input's shape, dtype and device")
    return out


def _drop(p: float, seed: int, offset: int, device_offset: torch.Tensor | None, dev: int) -> tuple:
    """The fields of mtxc_dropout_state."""
    at = 0
    if device_offset is not None:
        if device_offset.dtype not in (torch.int64, torch.uint64) or device_offset.numel() != 1 or \
                device_offset.get_device() != dev:
            raise ValueError("device_offset: expected one 64-bit integer on the tensors' device")
        at = device_offset.data_ptr()
    return float(p), seed & 0xFFFFFFFFFFFFFFFF, offset & 0xFFFFFFFFFFFFFFFF, at


# ------------------------------------------------------------------------------------------
# Operators
# ------------------------------------------------------------------------------------------
def dropout(x: torch.Tensor, p: float, seed: int, offset: int, *, device_offset: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """x with elements dropped with probability p and the others divided by 1 - p (both to 16 bits), by the
    counter-based generator of mtxc_dropout.  With the same seed and offset it is its own backward pass
    (gradients for x); every call of a step needs an offset of its own.  device_offset: one 64-bit integer on
    the device, added to offset when the kernel runs.  out may be x."""
    dev = _on_device(x)
    code = dtype_code(x.dtype)
    state = _abi.DROPOUT_STATE.pack(*_drop(p, seed, offset, device_offset, dev))
    out = _like(x, out, "out", dev)
    n = x.numel()
    if n == 0:
        return out
    width = x.shape[-1] if x.dim() else 1
    if out.is_contiguous() and x.is_contiguous():
        xs = os = width
    else:
        xs, os = _row_stride(x, "x"), _row_stride(out, "out", True)
    check(lib().mtxc_dropout(code, out.data_ptr(), x.data_ptr(), n // width, width, os, xs, state))
    return out


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


def _weight(w: torch.Tensor | None, width: int, what: str) -> int:
    if w is None:
        return 0
    if w.dim() != 1 or w.shape[0] != width or (width > 1 and w.stride(0) != 1):
        raise ValueError(f"{what}: expected {width} contiguous values")
    return w.data_ptr()


def _weight_dtype(a: torch.Tensor | None, b: torch.Tensor | None) -> int:
    if a is None:
        return dtype_code(b.dtype) if b is not None else 0
    if b is not None and a.dtype != b.dtype:
        raise ValueError("post_weight and next_weight: expected one dtype")
    return dtype_code(a.dtype)


def _gate(gate: torch.Tensor | None, x: torch.Tensor, rows: int) -> tuple[int, int, int, int]:
    """Pointer, row stride and dtype of the gate, and how many consecutive rows of x share a row of it: its
    leading axes are x's up to one, then ones."""
    if gate is None:
        return 0, 0, 0, 0
    if gate.dim() == 0 or gate.shape[-1] != x.shape[-1] or gate.dim() > x.dim():
        raise ValueError("gate: expected the rows' width and at most their axes")
    own, lead = tuple(gate.shape[:-1]), tuple(x.shape[:-1])
    share = max(1, rows)
    if any(n != 1 for n in own):
        share, i = 1, len(own)
        while own[i - 1] == 1:
            i -= 1
        if len(own) != len(lead) or own[:i] != lead[:i]:
            raise ValueError("gate: expected one row, or the leading axes with the last ones of extent 1")
        for n in lead[i:]:
            share *= n
    return gate.data_ptr(), _row_stride(gate, "gate"), dtype_code(gate.dtype), max(1, share)


def _same(t: torch.Tensor | None, x: torch.Tensor, what: str) -> None:
    if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
        raise ValueError(f"{what}: expected the residual's shape and dtype")


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
    dev = _on_device(residual, branch, post_weight, gate, next_weight)
    code = dtype_code(residual.dtype)
    _same(branch, residual, "branch")
    if residual.dim() == 0:
        raise ValueError("residual: expected rows")
    width = residual.shape[-1]
    rows = residual.numel() // width if width else 0
    if branch is None and (post_weight is not None or gate is not None):
        raise ValueError("post_weight and gate need a branch")
    h, h_ptr, h_stride = residual, 0, 0
    if branch is not None or residual_scale != 1.0 or out is not None:
        h = _like(residual, out, "out", dev)
        h_ptr, h_stride = h.data_ptr(), _row_stride(h, "out", True)
    a, a_ptr, a_stride = None, 0, 0
    if next_weight is not None:
        a = _like(residual, normed_out, "normed_out", dev)
        a_ptr, a_stride = a.data_ptr(), _row_stride(a, "normed_out", True)
    elif normed_out is not None:
        raise ValueError("normed_out needs next_weight")
    post_rstd = next_rstd = None
    if save_rstd:
        if post_weight is not None:
            post_rstd = _new(residual, (rows,), torch.float32, dev)
        if next_weight is not None:
            next_rstd = _new(residual, (rows,), torch.float32, dev)
    g_ptr, g_stride, g_code, g_rows = _gate(gate, residual, rows)
    check(lib().mtxc_block_norm(code, _abi.BLOCK_NORM_ARGS.pack(
        rows, width, residual.data_ptr(), _row_stride(residual, "residual"),
        branch.data_ptr() if branch is not None else 0, _row_stride(branch, "branch") if branch is not None else 0,
        _weight(post_weight, width, "post_weight"), _weight(next_weight, width, "next_weight"),
        g_ptr, g_stride, g_rows, h_ptr, h_stride, a_ptr, a_stride,
        post_rstd.data_ptr() if post_rstd is not None else 0, next_rstd.data_ptr() if next_rstd is not None else 0,
        _weight_dtype(post_weight, next_weight), g_code, residual_scale, branch_scale, weight_offset, eps, *_drop(dropout, seed, offset, device_offset, dev))))
    return BlockNorm(h, a, post_rstd, next_rstd)


def _rstd(t: torch.Tensor | None, rows: int, of: torch.Tensor | None, what: str) -> int:
    if of is None:
        return 0
    if t is None or t.dtype != torch.float32 or t.numel() != rows or not t.is_contiguous():
        raise ValueError(f"{what}: expected {rows} contiguous float32 values, as block_norm saves them")
    return t.data_ptr()


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
    dev = _on_device(residual, d_residual, d_normed, branch, post_rstd, next_rstd, post_weight, gate, next_weight)
    code = dtype_code(residual.dtype)
    _same(d_residual, residual, "d_residual")
    _same(d_normed, residual, "d_normed")
    _same(branch, residual, "branch")
    if residual.dim() == 0:
        raise ValueError("residual: expected rows")
    if (d_normed is None) != (next_weight is None):
        raise ValueError("d_normed and next_weight go together")
    if branch is None and (post_weight is not None or gate is not None):
        raise ValueError("post_weight and gate need a branch")
    width = residual.shape[-1]
    rows = residual.numel() // width if width else 0
    dx = _new(residual, residual.shape, residual.dtype, dev)
    db = _new(residual, residual.shape, residual.dtype, dev) if branch is not None else None
    dp = _new(residual, (width,), torch.float32, dev) if parameters and post_weight is not None else None
    dn = _new(residual, (width,), torch.float32, dev) if parameters and next_weight is not None else None
    dg = _new(gate, gate.shape, gate.dtype, dev) if parameters and gate is not None else None
    if rows == 0 and dg is not None:  # a sum over no rows (the call itself knows of no gate row then)
        check(lib().mtxc_memset(dg.data_ptr(), 0, dg.numel() * dg.element_size()))

    def at(t):
        return t.data_ptr() if t is not None else 0

    def stride(t, what):
        return _row_stride(t, what) if t is not None else 0

    g_ptr, g_stride, g_code, g_rows = _gate(gate, residual, rows)
    check(lib().mtxc_block_norm_backward(code, _abi.BLOCK_NORM_BACKWARD_ARGS.pack(
        rows, width, at(d_residual), stride(d_residual, "d_residual"), at(d_normed), stride(d_normed, "d_normed"),
        residual.data_ptr(), _row_stride(residual, "residual"), at(branch), stride(branch, "branch"),
        _rstd(post_rstd, rows, post_weight, "post_rstd"), _rstd(next_rstd, rows, next_weight, "next_rstd"),
        _weight(post_weight, width, "post_weight"), _weight(next_weight, width, "next_weight"), g_ptr,
        g_stride, g_rows, dx.data_ptr(), width, at(db), width, at(dp), at(dn), at(dg), width,
        _weight_dtype(post_weight, next_weight), g_code, residual_scale, branch_scale, weight_offset,
        *_drop(dropout, seed, offset, device_offset, dev))))
    return BlockNormGradients(dx, db, dp, dg, dn)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                       original_length: float = 0.0, fast_turns: float = 32.0, slow_turns: float = 1.0,
                       device="cuda") -> tuple[torch.Tensor, float]:
    """The frequencies (float64, rotary_dim / 2 of them, on the device) and the scale that `rotary` takes, for
    a context `factor` times as long as the one trained on: scaling "none", "linear", "base" or "by_parts"
    (mtxc_rotary_frequencies states them)."""
    values = (ctypes.c_double * max(1, rotary_dim // 2))()
    scale = ctypes.c_double()
    if scaling not in _abi.ROTARY_SCALINGS:
        raise ValueError(f"scaling: expected one of {sorted(_abi.ROTARY_SCALINGS)}")
    check(lib().mtxc_rotary_frequencies(_abi.ROTARY_SCALINGS[scaling], rotary_dim, base, factor, original_length,
                                        fast_turns, slow_turns, values, ctypes.byref(scale)))
    return torch.tensor(values[:rotary_dim // 2], dtype=torch.float64, device=device), scale.value


def _heads(x: torch.Tensor | None, out: torch.Tensor | None, what: str, dev: int):
    """A tensor of heads, what it is written to, and the two's strides over batch, length and heads."""
    if x is None:
        return None, 0, 0, 0, (0, 0, 0), (0, 0, 0)
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"{what}: the last axis needs unit stride")
    if out is None:
        if _own_memory(dev):
            out = torch.empty_like(x)
        else:
            with _on_stream(dev):
                out = torch.empty_like(x)
    elif out.shape != x.shape or out.dtype != x.dtype or out.get_device() != dev:
        raise ValueError(f"{what}'s output: expected its shape, dtype and device")
    elif out.shape[-1] > 1 and out.stride(-1) != 1:
        raise ValueError(f"{what}'s output: the last axis needs unit stride")
    xs, os = x.stride()[:-1], out.stride()[:-1]
    if x.dim() == 3:
        xs, os = (0, *xs), (0, *os)
    return out, x.shape[-2], out.data_ptr(), x.data_ptr(), os, xs


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, frequencies: torch.Tensor, *,
           scale: float = 1.0, interleaved: bool = False, inverse: bool = False,
           out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Queries and keys turned by their positions (mtxc_rotary), in one launch: q and k are [batch, length,
    heads, head_dim] or [length, heads, head_dim] with any strides (heads may be stored before tokens) but unit
    stride within a head; k may have fewer heads, or be None.  positions: int32 or int64, [batch, length] or
    [length].  frequencies and scale: as rotary_frequencies gives them; the first 2 * len(frequencies) elements
    of a head are turned, in pairs (j, j + half) or, interleaved, (2j, 2j + 1), and the others passed on.
    inverse=True is the backward pass.  out=(q, k) writes in place."""
    dev = _on_device(q, k, positions, frequencies)
    code = dtype_code(q.dtype)
    if q.dim() not in (3, 4):
        raise ValueError("q: expected [batch, length, heads, head_dim] or [length, heads, head_dim]")
    if k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1] or
                          k.dtype != q.dtype):
        raise ValueError("k: expected q's batch, length, head_dim and dtype")
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64 or not frequencies.is_contiguous():
        raise ValueError("frequencies: expected contiguous float64 values")
    batch, length = (q.shape[0], q.shape[1]) if q.dim() == 4 else (1, q.shape[0])
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions: expected int32 or int64")
    if tuple(positions.shape) == (length,):
        ps = (0, positions.stride(0))
    elif q.dim() == 4 and positions.dim() == 2 and positions.shape[1] == length and positions.shape[0] in (1, batch):
        ps = (positions.stride(0) if positions.shape[0] == batch else 0, positions.stride(1))
    else:
        raise ValueError("positions: expected [batch, length] or [length]")
    q_out, q_heads, q_dst, q_src, q_ds, q_ss = _heads(q, out[0] if out is not None else None, "q", dev)
    k_out, k_heads, k_dst, k_src, k_ds, k_ss = _heads(k, out[1] if out is not None else None, "k", dev)
    check(lib().mtxc_rotary(code, _abi.ROTARY_ARGS.pack(
        batch, length, q.shape[-1], 2 * frequencies.shape[0], q_heads, k_heads, q_dst, k_dst, *q_ds, *k_ds, q_src,
        k_src, *q_ss, *k_ss, positions.data_ptr(), dtype_code(positions.dtype), *ps, frequencies.data_ptr(), scale,
        interleaved, inverse)))
    return q_out, k_out


def _per_row(t: torch.Tensor | None, rows: int, dtype: torch.dtype, what: str) -> int:
    if t is None:
        return 0
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != rows or (rows > 1 and t.stride(0) != 1):
        raise ValueError(f"{what}: expected {rows} contiguous {dtype} values")
    return t.data_ptr()


def _lists(t: torch.Tensor | None, rows: int, dtypes: tuple, what: str) -> tuple[int, int, int]:
    """Pointer, row stride (0: one list for all rows) and length of lists [rows, n] or [n]."""
    if t is None:
        return 0, 0, 0
    if t.dtype not in dtypes or t.dim() not in (1, 2) or (t.dim() == 2 and t.shape[0] not in (1, rows)) or             (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{what}: expected [rows, n] or [n] of {dtypes[0]} with unit stride along n")
    return t.data_ptr(), t.stride(0) if t.dim() == 2 and t.shape[0] == rows else 0, t.shape[-1]


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
    dev = _on_device(logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias_tokens, bias_values,
                     mask)
    code = dtype_code(logits.dtype)
    if logits.dim() != 2:
        raise ValueError("logits: expected [rows, vocab]")
    rows, vocab = logits.shape
    if tokens is None and not (lengths is prompt_lengths is repetition is frequency is presence is None):
        raise ValueError("penalties need the rows' tokens")
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values go together")
    t_ptr, t_stride, history = _lists(tokens, rows, (torch.int32,), "tokens")
    b_ptr, b_stride, biases = _lists(bias_tokens, rows, (torch.int32,), "bias_tokens")
    v_ptr, v_stride, values = _lists(bias_values, rows, (torch.float32,), "bias_values")
    m_ptr, m_stride, words = _lists(mask, rows, (torch.int32, torch.uint32), "mask")
    if values != biases:
        raise ValueError("bias_values: expected one for each of bias_tokens")
    if mask is not None and words != (vocab + 31) // 32:
        raise ValueError("mask: expected one bit for each token, in words of 32")
    out = _like(logits, out, "out", dev)
    check(lib().mtxc_logits_rules(code, _abi.LOGITS_ARGS.pack(
        rows, vocab, out.data_ptr(), _row_stride(out, "out", True), logits.data_ptr(), _row_stride(logits, "logits"), t_ptr,
        t_stride, history, _per_row(lengths, rows, torch.int32, "lengths"),
        _per_row(prompt_lengths, rows, torch.int32, "prompt_lengths"),
        _per_row(repetition, rows, torch.float32, "repetition"), _per_row(frequency, rows, torch.float32, "frequency"),
        _per_row(presence, rows, torch.float32, "presence"), b_ptr, b_stride, v_ptr, v_stride, biases, m_ptr, m_stride)))
    return out
