"""The choice of the next token: temperature, top-k, top-p and min-p on a row of logits
with a given random number (``ossm_sample_logits``).

It is what ``control_logits`` leaves to do: both take a batch of requests, each with
settings of its own, in one launch and without the host looking at a value.
"""

from __future__ import annotations

from typing import Optional, Union

import torch
from torch import Tensor

from . import _lib

__all__ = ["sample_logits"]

_PerRow = Union[float, Tensor, None]


def _setting(v: _PerRow, rows: int, none: float, name: str, dev: int):
    """A setting as a float32 tensor of each row's, or as one number."""
    if v is None or isinstance(v, (int, float)):
        return None, none if v is None else float(v)
    if not isinstance(v, Tensor) or v.dtype != torch.float32 or v.shape != (rows,) or v.get_device() != dev:
        got = f"{v.dtype} {tuple(v.shape)} on {v.device}" if isinstance(v, Tensor) else type(v).__name__
        raise RuntimeError(f"sample_logits: {name} must be a number or a float32 tensor ({rows},) on the logits' GPU, got {got}")
    return v.contiguous(), none


def sample_logits(logits: Tensor, uniform: Tensor, *, temperature: _PerRow = None, top_k: Union[int, Tensor, None] = None,
                  top_p: _PerRow = None, min_p: _PerRow = None, out: Optional[Tensor] = None) -> Tensor:
    """A token of each row of logits [rows, V] (float32 or bfloat16), int64 [rows], drawn by
    the random numbers ``uniform`` (float32 [rows], in [0, 1)) from softmax(logits /
    temperature) after, in this order,

    * ``top_k``: the k largest logits are kept (0 or less: all);
    * ``top_p``: of those, in falling order, each before which less than p of their
      probability lies (1 or more: all);
    * ``min_p``: of those, each of at least ``min_p`` times the most likely one's probability.

    The most likely token is always kept; of equal logits the lower index comes first.  The
    token is the first, by index, at which the kept probabilities' running sum passes
    ``uniform`` times their sum.  A temperature that is not above 0 answers the most likely
    token.  Each setting is a number or a float32 (top_k: int32 or int64) tensor [rows]; numbers are taken as
    float32.  NaN counts as -inf, +inf shares the answer with its like; a row of which
    nothing is above -inf (a mask that allows nothing) answers -1.  ``out`` (int64 [rows], any
    stride) takes the result.  The sums are of whole numbers in 64 bits: the answer is the exact
    one, but for weights below 2^-43 of the largest.  V is at most 2^20.  Nothing synchronises; a
    call may be captured in a HIP graph.  The result carries no gradient."""
    dev = logits.get_device()
    if logits.dtype not in _lib.LM_DTYPES or dev < 0 or logits.dim() != 2:
        raise RuntimeError("sample_logits: logits must be a float32 or bfloat16 GPU tensor (rows, vocabulary), got "
                           f"{logits.dtype} {tuple(logits.shape)} on {logits.device}")
    rows, V = logits.shape
    if uniform.dtype != torch.float32 or uniform.shape != (rows,) or uniform.get_device() != dev:
        raise RuntimeError(f"sample_logits: uniform must be a float32 tensor ({rows},) on the logits' GPU, got {uniform.dtype} "
                           f"{tuple(uniform.shape)} on {uniform.device}")
    if not 0 < V <= 1 << 20:
        raise RuntimeError(f"sample_logits: the vocabulary must have 1 to 2^20 tokens, got {V}")
    temperature, t_all = _setting(temperature, rows, 1.0, "temperature", dev)
    top_p, p_all = _setting(top_p, rows, 1.0, "top_p", dev)
    min_p, m_all = _setting(min_p, rows, 0.0, "min_p", dev)
    k_all = 0
    if top_k is not None and not isinstance(top_k, Tensor):
        k_all, top_k = min(max(int(top_k), 0), 2**31 - 1), None
    elif top_k is not None:
        if top_k.dtype not in (torch.int32, torch.int64) or top_k.shape != (rows,) or top_k.get_device() != dev:
            raise RuntimeError(f"sample_logits: top_k must be a number or an int32 or int64 tensor ({rows},) on the logits' GPU, "
                               f"got {top_k.dtype} {tuple(top_k.shape)} on {top_k.device}")
        # a count past int32 would wrap
        top_k = (top_k if top_k.dtype == torch.int32 else top_k.clamp(0, 2**31 - 1).to(torch.int32)).contiguous()
    if out is None:
        tokens = torch.empty((rows,), dtype=torch.int64, device=logits.device)
    elif out.dtype != torch.int64 or out.shape != (rows,) or out.get_device() != dev:
        raise RuntimeError(f"sample_logits: out must be an int64 tensor ({rows},) on the logits' GPU, got {out.dtype} "
                           f"{tuple(out.shape)} on {out.device}")
    else:
        tokens = out if out.is_contiguous() else torch.empty((rows,), dtype=torch.int64, device=logits.device)
    if V > 1 and (logits.stride(1) != 1 or logits.stride(0) < 0):
        logits = logits.contiguous()
    uniform = uniform.contiguous()
    _lib.run(_lib.load().ossm_sample_logits, logits, _lib.LM_DTYPES[logits.dtype], logits.data_ptr(), logits.stride(0),
             uniform.data_ptr(), _lib.ptr(temperature), t_all, _lib.ptr(top_k), k_all, _lib.ptr(top_p), p_all,
             _lib.ptr(min_p), m_all, tokens.data_ptr(), rows, V)
    if out is not None and tokens is not out:
        out.copy_(tokens)
        return out
    return tokens
