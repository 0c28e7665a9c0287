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

_pack = _lib.words_of("grs_adjust_logits").pack
_entry = None


def _ints(name: str, t: torch.Tensor | None, rows: int, device: int) -> int:
    """Address of an optional int32 [rows], or 0."""
    if t is None:
        return 0
    if (t.dtype is not torch.int32 or t.shape != (rows,) or not t.is_contiguous()
            or t.get_device() != device):
        _lib.require_cuda(t)
        raise ValueError(f"{name} must be contiguous int32 [rows] on the logits' device")
    return t.data_ptr()


def _knob(name: str, value, rows: int, device: int):
    """(address or 0, scalar) of a penalty given per row or for all."""
    if isinstance(value, torch.Tensor):
        if (value.dtype is not torch.float32 or value.shape != (rows,)
                or not value.is_contiguous() or value.get_device() != device):
            _lib.require_cuda(value)
            raise ValueError(f"{name} must be a number or contiguous fp32 [rows]")
        return value.data_ptr(), 0.0
    return 0, float(value)


def _table(name: str, t: torch.Tensor, dtype: torch.dtype, rows: int, columns: int,
           device: int) -> int:
    """Row stride of a [columns], [1, columns] or [rows, columns] tensor."""
    shape, stride = t.shape, t.stride()
    if (t.dtype is not dtype or t.get_device() != device or not 1 <= len(shape) <= 2
            or shape[-1] != columns or (len(shape) == 2 and shape[0] not in (1, rows))
            or (columns > 1 and stride[-1] != 1)):
        _lib.require_cuda(t)
        raise ValueError(f"{name} must be {dtype} [{columns}] or [{rows}, {columns}] with "
                         "contiguous rows on the logits' device")
    return stride[0] if len(shape) == 2 and shape[0] > 1 else 0


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
    or ``out`` (``out=logits`` adjusts in place; otherwise it must not overlap
    them, and never the other inputs).

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
    global _entry
    device = logits.get_device()
    if device < 0:
        _lib.require_cuda(logits)
    place = _lib.elsewhere(device)
    if place is not None:
        with place:
            return adjust_logits(logits, tokens=tokens, lengths=lengths,
                                 prompt_lengths=prompt_lengths, repetition=repetition,
                                 presence=presence, frequency=frequency, bias=bias,
                                 allowed=allowed, fill=fill, out=out)
    dtype = logits.dtype
    code = _lib.DTYPE_CODES.get(dtype)
    if code is None or logits.dim() != 2:
        raise ValueError("logits must be bf16 or fp32 [rows, vocab]")
    rows, vocab = logits.shape
    if rows >= 1 << 30 or vocab >= 1 << 30:
        raise ValueError("at most 2^30 rows and columns")
    row, step = logits.stride()
    if vocab > 1 and step != 1:
        raise ValueError("logits need contiguous rows")
    history = tokens_row = wide = 0
    token_ptr = 0
    if tokens is not None:
        if (tokens.dtype not in (torch.int32, torch.int64) or tokens.dim() != 2
                or tokens.shape[0] != rows or tokens.get_device() != device
                or (tokens.shape[1] > 1 and tokens.stride(1) != 1)):
            _lib.require_cuda(tokens)
            raise ValueError("tokens must be int32 or int64 [rows, history], contiguous rows")
        history, tokens_row = tokens.shape[1], tokens.stride(0)
        if history >= 1 << 30:
            raise ValueError("histories hold at most 2^30 tokens")
        wide, token_ptr = int(tokens.dtype is torch.int64), tokens.data_ptr()
    elif lengths is not None or prompt_lengths is not None:
        raise ValueError("lengths and prompt_lengths come with tokens")
    lengths_ptr = _ints("lengths", lengths, rows, device)
    prompts_ptr = _ints("prompt_lengths", prompt_lengths, rows, device)
    rep_ptr, rep = _knob("repetition", repetition, rows, device)
    pres_ptr, pres = _knob("presence", presence, rows, device)
    freq_ptr, freq = _knob("frequency", frequency, rows, device)
    if not rep_ptr and not rep > 0:
        raise ValueError("repetition must be positive")
    bias_ptr = allowed_ptr = 0
    bias_row = allowed_row = 0
    if bias is not None:
        bias_row = _table("bias", bias, torch.float32, rows, vocab, device)
        bias_ptr = bias.data_ptr()
    if allowed is not None:
        allowed_row = _table("allowed", allowed, torch.int32, rows, (vocab + 31) // 32, device)
        allowed_ptr = allowed.data_ptr()
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
        out_row = vocab
    else:
        if (out.shape != logits.shape or out.dtype is not dtype or out.get_device() != device
                or (vocab > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < vocab)):
            _lib.require_cuda(out)
            raise ValueError("out must have the logits' shape, dtype and device, contiguous rows")
        out_row = out.stride(0)
        if rows > 1 and out_row != row and out.data_ptr() == logits.data_ptr():
            raise ValueError("out must be the logits themselves or not overlap them")
        if bias_ptr == out.data_ptr() and bias is not None and out.numel():
            raise ValueError("out must not be the bias")
    if not rows or not vocab:
        return out
    if _entry is None:
        _entry = _lib.words_entry("grs_adjust_logits")
    status = _entry(_pack(
        code, logits.data_ptr(), row, out.data_ptr(), out_row, rows, vocab, token_ptr, wide,
        tokens_row, history, lengths_ptr, prompts_ptr, rep_ptr, pres_ptr, freq_ptr, rep, pres,
        freq, bias_ptr, bias_row, allowed_ptr, allowed_row, float(fill),
        _lib.stream_on(device)))
    if status:
        _lib.check(status, "adjust_logits")
    return out
