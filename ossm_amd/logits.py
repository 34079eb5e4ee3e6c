"""Control of the logits a model answers with: penalties for repeated tokens, biases
and a grammar's mask, in one pass (``ossm_control_logits``)."""

from __future__ import annotations

from typing import Optional, Union

import torch
from torch import Tensor

from . import _lib

__all__ = ["control_logits", "pack_allowed"]

_PerRow = Union[float, Tensor, None]


def pack_allowed(allowed: Tensor) -> Tensor:
    """A bool mask [..., V] (True: the token may be answered) as the int32 words
    [..., ceil(V / 32)] that ``control_logits`` takes, token v in bit v % 32 of word
    v // 32."""
    V = allowed.size(-1)
    a = torch.nn.functional.pad(allowed.to(torch.int64), (0, -V % 32)).unflatten(-1, (-1, 32))
    w = (a << torch.arange(32, device=a.device)).sum(-1)
    return torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)


def _rows(t: Optional[Tensor], rows: int, cols: Optional[int], dtype: torch.dtype, name: str, dev: int):
    """A [rows, cols] tensor (or None) with unit column stride, and its row stride; one
    row may stand for all."""
    if t is None:
        return None, 0
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if t.dim() != 2 or t.size(0) not in (1, rows) or (cols is not None and t.size(1) != cols) or t.dtype != dtype \
            or t.get_device() != dev:
        raise RuntimeError(f"control_logits: {name} must be a {dtype} tensor ({rows}, {'*' if cols is None else cols}) on "
                           f"the logits' GPU, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.stride(1) != 1 and t.size(1) > 1:
        t = t.contiguous()
    return t, (t.stride(0) if t.size(0) > 1 else 0)


def _per_row(v: _PerRow, rows: int, none: float, name: str, dev: int):
    """A per-row float32 tensor, or a number for every row."""
    if v is None or isinstance(v, (int, float)):
        return None, none if v is None else float(v)
    if v.dtype != torch.float32 or v.shape != (rows,) or v.get_device() != dev:
        raise RuntimeError(f"control_logits: {name} must be a number or a float32 tensor ({rows},) on the logits' GPU, "
                           f"got {v.dtype} {tuple(v.shape)} on {v.device}")
    return v.contiguous(), none


def _lengths(t: Optional[Tensor], rows: int, name: str, dev: int) -> Optional[Tensor]:
    if t is None:
        return None
    if t.dtype not in (torch.int32, torch.int64) or t.shape != (rows,) or t.get_device() != dev:
        raise RuntimeError(f"control_logits: {name} must be an int32 or int64 tensor ({rows},) on the logits' GPU, got "
                           f"{t.dtype} {tuple(t.shape)} on {t.device}")
    # a length past int32 would wrap
    return (t if t.dtype == torch.int32 else t.clamp(0, 2**31 - 1).to(torch.int32)).contiguous()


def control_logits(logits: Tensor, history: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                   prompt_lengths: Optional[Tensor] = None, *, repetition: _PerRow = None, presence: _PerRow = None,
                   frequency: _PerRow = None, bias_ids: Optional[Tensor] = None, bias_values: Optional[Tensor] = None,
                   allowed: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """logits [rows, V] (float32 or bfloat16) after, in this order,

    * ``repetition``: a token of ``history[:length]`` has its logit divided by it where
      positive and multiplied by it elsewhere;
    * ``frequency`` times the token's count in ``history[prompt_length:length]`` and
      ``presence``, once, for one that occurs there, subtracted;
    * ``bias_values[j]`` added to token ``bias_ids[j]`` (of an id given twice the last
      counts);
    * -inf wherever ``allowed`` (``pack_allowed``) has no bit, whatever the logit was.

    history int32 [rows, H] of token ids, of which a row's first ``lengths`` (default H)
    count and the first ``prompt_lengths`` (default 0) are the prompt; bias_ids int32,
    bias_values float32 [rows, n]; ids outside the vocabulary are padding.  The three
    penalties are numbers or float32 tensors [rows]; history, biases and allowed may
    have one row for all.  A row whose mask allows nothing is all -inf.  ``out``
    (``logits`` itself to work in place) takes the result, else a new tensor; it is
    computed in float32 and rounded once.  Inference only: a call that would need a
    gradient or carries a forward-mode tangent raises."""
    dev = logits.get_device()
    if logits.dtype not in _lib.LM_DTYPES or dev < 0 or logits.dim() != 2:
        raise RuntimeError("control_logits: logits must be a float32 or bfloat16 GPU tensor (rows, vocabulary), got "
                           f"{logits.dtype} {tuple(logits.shape)} on {logits.device}")
    rows, V = logits.shape
    given = (logits, repetition, presence, frequency, bias_values, out)
    needs_grad = torch.is_grad_enabled() and any(isinstance(t, Tensor) and t.requires_grad for t in given)
    if needs_grad or _lib.has_tangent(given):
        raise RuntimeError("control_logits is for inference: call it under torch.no_grad() and on tensors without tangents")
    if (bias_ids is None) != (bias_values is None):
        raise RuntimeError("control_logits: give both bias_ids and bias_values, or neither")
    if history is None and (lengths is not None or prompt_lengths is not None):
        raise RuntimeError("control_logits: lengths without a history")
    if history is not None and history.dim() != 2:  # one token of each row would pass for one row's history
        raise RuntimeError(f"control_logits: history must be (rows, tokens) or (1, tokens), got {tuple(history.shape)}")
    history, ld_h = _rows(history, rows, None, torch.int32, "history", dev)
    lengths, prompt_lengths = (_lengths(lengths, rows, "lengths", dev),
                               _lengths(prompt_lengths, rows, "prompt_lengths", dev))
    rep, rep_all = _per_row(repetition, rows, 1.0, "repetition", dev)
    pres, pres_all = _per_row(presence, rows, 0.0, "presence", dev)
    freq, freq_all = _per_row(frequency, rows, 0.0, "frequency", dev)
    bias_ids, ld_b = _rows(bias_ids, rows, None, torch.int32, "bias_ids", dev)
    n_bias = 0 if bias_ids is None else bias_ids.size(1)
    if bias_values is not None:
        bias_values, ld_v = _rows(bias_values, rows, n_bias, torch.float32, "bias_values", dev)
        if ld_v != ld_b:  # one row stride for both
            bias_ids, bias_values = (t.expand(rows, n_bias).contiguous() for t in (bias_ids, bias_values))
            ld_b = n_bias
    allowed, ld_a = _rows(allowed, rows, (V + 31) // 32, torch.int32, "allowed", dev)
    if out is None:
        out = torch.empty((rows, V), dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.get_device() != dev or \
            (V > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < V):
        raise RuntimeError("control_logits: out must have the logits' shape, dtype and device and whole rows, got "
                           f"{out.dtype} {tuple(out.shape)} strides {out.stride()} on {out.device}")
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    _lib.run(_lib.load().ossm_control_logits, logits, _lib.LM_DTYPES[logits.dtype], logits.data_ptr(),
             logits.stride(0), out.data_ptr(), out.stride(0), _lib.ptr(history), ld_h,
             0 if history is None else history.size(1), _lib.ptr(lengths), _lib.ptr(prompt_lengths), _lib.ptr(rep),
             rep_all, _lib.ptr(pres), pres_all, _lib.ptr(freq), freq_all, _lib.ptr(bias_ids), _lib.ptr(bias_values),
             ld_b, n_bias, _lib.ptr(allowed), ld_a, rows, V)
    return out
