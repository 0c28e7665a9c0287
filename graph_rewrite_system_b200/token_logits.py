"""Next-token logits before ranking: penalties for repeated tokens, biases and
grammar masks.

``match_logits`` masks rewrite sources that a slot cannot match;
``adjust_logits`` is the counterpart for a token vocabulary, one launch over
the logits of every beam.  Inference only: no gradient is recorded.  The
sm_100a kernel lives in ``csrc/token_logits.cu``; CPU tensors raise.
"""
from __future__ import annotations

import torch

from . import _lib


def _knob(name: str, value, rows: int, device: torch.device):
    """(device pointer or None, scalar) of a penalty given per row or for all."""
    if isinstance(value, torch.Tensor):
        _lib.require_cuda(value)
        if (value.dtype != torch.float32 or tuple(value.shape) != (rows,)
                or not value.is_contiguous() or value.device != device):
            raise ValueError(f"{name} must be a number or contiguous fp32 [rows]")
        return value.data_ptr(), 0.0
    return None, float(value)


def _row_stride(name: str, t: torch.Tensor, rows: int, columns: int, device) -> int:
    """Row stride of a [columns], [1, columns] or [rows, columns] tensor."""
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if t.dim() != 2 or t.shape[0] not in (1, rows) or t.shape[1] != columns:
        raise ValueError(f"{name} must be [{columns}] or [{rows}, {columns}]")
    if t.device != device or (columns > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} needs contiguous rows on the logits' device")
    return t.stride(0) if t.shape[0] > 1 else 0


def adjust_logits(
    logits: torch.Tensor,
    *,
    tokens: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    prompt_lengths: torch.Tensor | None = None,
    repetition: float | torch.Tensor = 1.0,
    presence: float | torch.Tensor = 0.0,
    frequency: float | torch.Tensor = 0.0,
    bias: torch.Tensor | None = None,
    allowed: torch.Tensor | None = None,
    fill: float = float("-inf"),
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Adjusted copy of logits [rows, vocab] (bf16 or fp32, contiguous rows),
    or ``out`` (``out=logits`` adjusts in place).

    For every token v of row b, in this order: if v is among the first
    ``lengths[b]`` (default: all) of ``tokens[b]`` (int32 or int64 [rows,
    history]; ids outside the vocabulary are ignored, so any of them pads), x
    becomes ``x / repetition`` where it is positive and ``x * repetition``
    elsewhere; if v occurs c > 0 times among them from ``prompt_lengths[b]``
    (default 0) on, ``frequency * c + presence`` is subtracted; ``bias`` (fp32
    [vocab] or [rows, vocab]) is added; x becomes ``fill`` where bit ``v % 32``
    of ``allowed[b, v // 32]`` (int32 [words] or [rows, words], words =
    ceil(vocab / 32)) is clear, whatever it held.  A row whose mask leaves
    nothing is all ``fill``.  repetition (> 0), presence and frequency are
    numbers or fp32 [rows].  Computed in fp32 and rounded once.
    """
    _lib.require_cuda(logits, tokens, lengths, prompt_lengths, bias, allowed, out)
    if logits.dtype not in _lib.DTYPE_CODES or logits.dim() != 2:
        raise ValueError("logits must be bf16 or fp32 [rows, vocab]")
    rows, vocab = logits.shape
    device = logits.device
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("logits need contiguous rows")
    history = 0
    if tokens is not None:
        if (tokens.dtype not in (torch.int32, torch.int64) or tokens.dim() != 2
                or tokens.shape[0] != rows or tokens.device != device
                or (tokens.shape[1] > 1 and tokens.stride(1) != 1)):
            raise ValueError("tokens must be int32 or int64 [rows, history], contiguous rows")
        history = tokens.shape[1]
    elif lengths is not None or prompt_lengths is not None:
        raise ValueError("lengths and prompt_lengths come with tokens")
    for name, t in (("lengths", lengths), ("prompt_lengths", prompt_lengths)):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (rows,)
                              or not t.is_contiguous() or t.device != device):
            raise ValueError(f"{name} must be contiguous int32 [rows]")
    rep_ptr, rep = _knob("repetition", repetition, rows, device)
    pres_ptr, pres = _knob("presence", presence, rows, device)
    freq_ptr, freq = _knob("frequency", frequency, rows, device)
    if rep_ptr is None and not rep > 0:
        raise ValueError("repetition must be positive")
    bias_sb = allowed_sb = 0
    if bias is not None:
        if bias.dtype != torch.float32:
            raise ValueError("bias must be fp32")
        bias_sb = _row_stride("bias", bias, rows, vocab, device)
    if allowed is not None:
        if allowed.dtype != torch.int32:
            raise ValueError("allowed must be int32 words")
        allowed_sb = _row_stride("allowed", allowed, rows, -(-vocab // 32), device)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=device)
    elif (out.shape != logits.shape or out.dtype != logits.dtype or out.device != device
          or (vocab > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < vocab)):
        raise ValueError("out must have the logits' shape, dtype and device, contiguous rows")
    elif out.data_ptr() == logits.data_ptr() and rows > 1 and out.stride(0) != logits.stride(0):
        raise ValueError("out must be the logits themselves or not overlap them")
    if not logits.numel():
        return out
    with _lib.on_device(logits):
        code = _lib.lib().grs_adjust_logits(
            _lib.DTYPE_CODES[logits.dtype], logits.data_ptr(), logits.stride(0), out.data_ptr(),
            out.stride(0), rows, vocab, _lib.ptr(tokens),
            int(tokens is not None and tokens.dtype == torch.int64),
            0 if tokens is None else tokens.stride(0), history, _lib.ptr(lengths),
            _lib.ptr(prompt_lengths), rep_ptr, pres_ptr, freq_ptr, rep, pres, freq,
            _lib.ptr(bias), bias_sb, _lib.ptr(allowed), allowed_sb, float(fill),
            _lib.stream_of(logits))
    _lib.check(code, "adjust_logits")
    return out
