"""The gated projection of a feed-forward block, ``act(x Wg^T + bg) * (x Wu^T + bu)``,
forward and backward in this library's matrix-core kernels (``ossm_gated_forward``,
``ossm_gated_backward``), and the block built on it.

A block of the reference's backbones ends in such a gate (the GLU of
``ResidualSSMBlock``, base.py:113-155, with a sigmoid); a language model puts one,
with a down projection, after each mixer.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from . import _lib
from .linear import aliases, is_linear, linear

__all__ = ["ACTIVATIONS", "GatedFeedForward", "GatedLinearFn", "gated_linear"]

# the C ABI's numbers
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "sigmoid": 3, "relu": 4}

_TORCH = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"),
          "sigmoid": torch.sigmoid, "relu": F.relu}


def _separate(x: Tensor, wg: Tensor, wu: Tensor, bg: Optional[Tensor], bu: Optional[Tensor], act: str) -> Tensor:
    """The projection as torch's separate steps."""
    return _TORCH[act](F.linear(x, wg, bg)) * F.linear(x, wu, bu)


def _matrix(t: Tensor) -> Tensor:
    """``t`` itself where its rows are whole and do not overlap, else a dense copy (of rows
    broadcast from one, too, where they are single columns)."""
    rows, cols = t.shape
    return t if (cols <= 1 or t.stride(1) == 1) and (rows <= 1 or max(cols, 1) <= t.stride(0) <= 1 << 20) \
        else t.contiguous()


def _ld(t: Tensor) -> int:
    """The row stride of such a matrix (where nothing is read at it, any that holds a row)."""
    return max(t.stride(0), t.size(1)) if t.size(0) > 1 and t.size(1) > 0 else t.size(1)


def _forward(x: Tensor, wg: Tensor, wu: Tensor, bg: Optional[Tensor], bu: Optional[Tensor], act: str, save: bool):
    T, D, n = x.size(0), x.size(1), wg.size(0)
    x, wg, wu = _matrix(x), _matrix(wg), _matrix(wu)
    bg, bu = (None if b is None else b.contiguous() for b in (bg, bu))
    y = torch.empty((T, n), dtype=x.dtype, device=x.device)
    a, b = (torch.empty((T, n), dtype=torch.float32, device=x.device) if save else None for _ in range(2))
    if y.numel() > 0:
        _lib.run(_lib.load().ossm_gated_forward, x, _lib.LM_DTYPES[x.dtype], x.data_ptr(), _ld(x), wg.data_ptr(), _ld(wg),
                 wu.data_ptr(), _ld(wu), _lib.ptr(bg), _lib.ptr(bu), ACTIVATIONS[act], y.data_ptr(), _lib.ptr(a),
                 _lib.ptr(b), T, D, n)
    return y, a, b


class GatedLinearFn(torch.autograd.Function):
    """``gated_linear`` on matrices; saves both projections' outputs, in float32."""

    @staticmethod
    def forward(ctx, x: Tensor, wg: Tensor, wu: Tensor, bg: Optional[Tensor], bu: Optional[Tensor], act: str):  # type: ignore[override]
        y, a, b = _forward(x, wg, wu, bg, bu, act, True)
        ctx.act = act
        ctx.save_for_backward(x, wg, wu, bg, bu, a, b)
        return y

    @staticmethod
    def backward(ctx, gy: Tensor):  # type: ignore[override]
        x, wg, wu, bg, bu, a, b = ctx.saved_tensors
        need = ctx.needs_input_grad
        if torch.is_grad_enabled():
            # create_graph: differentiable again, as separate steps
            inputs = aliases(x, wg, wu, bg, bu)
            wanted = [t for t, n in zip(inputs, need) if n]
            got = iter(torch.autograd.grad(_separate(*inputs, ctx.act), wanted, gy, create_graph=True))
            return (*(next(got) if n else None for n in need[:5]), None)
        x, wg, wu, gy = _matrix(x), _matrix(wg), _matrix(wu), _matrix(gy)
        T, D, n = x.size(0), x.size(1), wg.size(0)
        out = [torch.empty(s, dtype=x.dtype, device=x.device) if k else None
               for s, k in zip(((T, D), (n, D), (n, D), (n,), (n,)), need)]
        _lib.run(_lib.load().ossm_gated_backward, x, _lib.LM_DTYPES[x.dtype], gy.data_ptr(), _ld(gy), x.data_ptr(), _ld(x),
                 wg.data_ptr(), _ld(wg), wu.data_ptr(), _ld(wu), ACTIVATIONS[ctx.act], a.data_ptr(), b.data_ptr(),
                 *(_lib.ptr(t) for t in out), T, D, n)
        return (*out, None)


def gated_linear(x: Tensor, gate_weight: Tensor, up_weight: Tensor, gate_bias: Optional[Tensor] = None,
                 up_bias: Optional[Tensor] = None, activation: str = "silu") -> Tensor:
    """``act(x @ gate_weight.T + gate_bias) * (x @ up_weight.T + up_bias)`` for x
    [..., D] and weights [F, D] (as two ``nn.Linear`` hold them): float32 or bfloat16
    tensors of one dtype on one GPU, any strides.  activation: silu, gelu, gelu_tanh,
    sigmoid or relu.  Sums are float32, and float32 products keep its 24 bits; the
    result is rounded once.  Differentiable in every argument (in reverse mode; a
    forward-mode tangent raises), twice as torch's separate steps; training keeps the two projections' outputs in float32.  Under a bfloat16
    autocast, float32 arguments are cast as ``F.linear``'s are."""
    args = [x, gate_weight, up_weight, gate_bias, up_bias]
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated_linear: activation must be one of {', '.join(ACTIVATIONS)}, not {activation!r}")
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
        args = [t if t is None or t.dtype != torch.float32 else t.bfloat16() for t in args]
        x, gate_weight, up_weight, gate_bias, up_bias = args
    index = x.get_device()
    for t in args:
        if t is not None and (t.dtype != x.dtype or x.dtype not in _lib.LM_DTYPES or index < 0 or t.get_device() != index):
            raise RuntimeError("gated_linear: x, weights and biases must be float32 or bfloat16 tensors of one dtype on one "
                               f"GPU, got {[None if t is None else (t.dtype, str(t.device)) for t in args]}")
    D = x.size(-1) if x.dim() > 0 else -1
    n = gate_weight.size(0) if gate_weight.dim() == 2 else -1
    if D < 0 or gate_weight.shape != (n, D) or up_weight.shape != (n, D) or \
            any(b is not None and b.shape != (n,) for b in (gate_bias, up_bias)):
        raise RuntimeError("gated_linear: expected x (..., D), weights (F, D), biases (F,), got "
                           f"{[None if t is None else tuple(t.shape) for t in args]}")
    if _lib.has_tangent(args):
        raise RuntimeError("gated_linear has no forward-mode derivative, and an argument carries a tangent")
    x2 = x if x.dim() == 2 else x.reshape(-1, D) if D > 0 else x.reshape(x.shape[:-1].numel(), 0)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        y = GatedLinearFn.apply(x2, gate_weight, up_weight, gate_bias, up_bias, activation)
    else:
        y = _forward(x2, gate_weight, up_weight, gate_bias, up_bias, activation, False)[0]
    return y if x.dim() == 2 else y.view(*x.shape[:-1], n)


class GatedFeedForward(nn.Module):
    """``down(act(gate(x)) * up(x))``: a model's feed-forward block, both projections, the
    activation and the product in one kernel."""

    def __init__(self, d_model: int, d_hidden: int, *, activation: str = "silu", bias: bool = False) -> None:
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, not {activation!r}")
        self.activation = activation
        self.gate_proj = nn.Linear(d_model, d_hidden, bias=bias)
        self.up_proj = nn.Linear(d_model, d_hidden, bias=bias)
        self.down_proj = nn.Linear(d_hidden, d_model, bias=bias)

    def forward(self, x: Tensor) -> Tensor:
        if is_linear(self.gate_proj) and is_linear(self.up_proj):
            h = gated_linear(x, self.gate_proj.weight, self.up_proj.weight, self.gate_proj.bias, self.up_proj.bias,
                             self.activation)
        else:  # a replaced or hooked projection is called as it is
            h = _TORCH[self.activation](linear(self.gate_proj, x)) * linear(self.up_proj, x)
        return linear(self.down_proj, h)
