"""Layer norm, alone or of a residual sum, forward and backward in this library's kernels
(``ossm_layer_norm_forward``, ``ossm_layer_norm_backward``).

The reference's backbones and a language model's blocks add what a block computed to the
residual stream and norm the sum for the next block; ``add_layer_norm`` is both in one
pass, and its backward joins the two gradients that reach the sum.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from . import _lib
from .gated import _ld, _matrix
from .linear import aliases, calls_only

__all__ = ["LayerNorm", "LayerNormFn", "add_layer_norm", "layer_norm", "norm_of_sum"]


def _separate(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], bias: Optional[Tensor], eps: float):
    """The same as torch's separate steps."""
    s = x if residual is None else x + residual
    cast = [t if t is None or t.dtype == s.dtype else t.to(s.dtype) for t in (weight, bias)]
    if cast[0] is weight and cast[1] is bias:
        y = F.layer_norm(s, s.shape[-1:], weight, bias, eps)
    else:  # float32 weights are not rounded
        y = F.layer_norm(s.float(), s.shape[-1:], weight, bias, eps).to(s.dtype)
    return y if residual is None else (y, s)


def _dense_like(t: Tensor) -> Tensor:
    """An empty dense tensor as ``t``; a call with sizes, type and device takes a microsecond longer."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _rows(t: Tensor, D: int) -> Tuple[Tensor, int]:
    """``t`` [..., D], not empty, as rows and their stride: itself where it is dense (a reshape is a node of
    its own in training), else as a matrix."""
    if t.is_contiguous():
        return t, D
    t = _matrix(t.reshape(-1, D))
    return t, _ld(t)


def _forward(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], bias: Optional[Tensor], eps: float, save: bool):
    dtype, D = x.dtype, x.size(-1)
    T = x.numel() // D if D > 0 else 0
    y = _dense_like(x)
    s = None if residual is None else _dense_like(x)
    stats = torch.empty((2, T), dtype=torch.float32, device=x.device) if save else None  # mean, rstd
    if T > 0:
        (x, ld), (residual, ld_res) = _rows(x, D), (None, 0) if residual is None else _rows(residual, D)
        weight, bias = None if weight is None else weight.contiguous(), None if bias is None else bias.contiguous()
        wt = weight if weight is not None else bias
        mean = _lib.ptr(stats)
        _lib.run(_lib.load().ossm_layer_norm_forward, x, _lib.LM_DTYPES[dtype], _lib.LM_DTYPES[dtype if wt is None else wt.dtype],
                 x.data_ptr(), ld, _lib.ptr(residual), ld_res, _lib.ptr(weight), _lib.ptr(bias), eps, y.data_ptr(),
                 _lib.ptr(s), mean, None if mean is None else mean + 4 * T, T, D)
    return y, s, stats


class LayerNormFn(torch.autograd.Function):
    """``layer_norm`` and ``add_layer_norm``; saves the sum and two numbers a row."""

    @staticmethod
    def forward(ctx, x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], bias: Optional[Tensor],  # type: ignore[override]
                eps: float):
        y, s, stats = _forward(x, residual, weight, bias, eps, True)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if s is None else s, weight, bias, stats)
        return y if s is None else (y, s)

    @staticmethod
    def backward(ctx, gy: Optional[Tensor], gs: Optional[Tensor] = None):  # type: ignore[override]
        s, weight, bias, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        if gy is None:  # nothing reaches the norm, whose rows may be NaN
            return gs if need[0] else None, gs if need[1] else None, None, None, None
        if torch.is_grad_enabled():
            # create_graph: differentiable again, as separate steps on the sum
            inputs = aliases(s, weight, bias)
            wanted = [t for t, n in zip(inputs, (need[0] or need[1], *need[2:4])) if n]
            got = iter(torch.autograd.grad(_separate(inputs[0], None, *inputs[1:], ctx.eps), wanted, gy, create_graph=True))
            ds = next(got) if need[0] or need[1] else None
            if ds is not None and gs is not None:
                ds = ds + gs
            return (ds if need[0] else None, ds if need[1] else None, *(next(got) if n else None for n in need[2:4]), None)
        wt = weight if weight is not None else bias
        ds = _dense_like(s) if need[0] or need[1] else None
        dw, db = _dense_like(wt) if need[2] else None, _dense_like(wt) if need[3] else None
        if s.numel() == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        else:
            D = s.size(-1)
            T = s.numel() // D
            (s, ld), (gy, ld_gy), (gs, ld_gs) = _rows(s, D), _rows(gy, D), (None, 0) if gs is None else _rows(gs, D)
            weight = None if weight is None else weight.contiguous()
            mean = stats.data_ptr()
            _lib.run(_lib.load().ossm_layer_norm_backward, s, _lib.LM_DTYPES[s.dtype],
                     _lib.LM_DTYPES[(s if wt is None else wt).dtype], gy.data_ptr(), ld_gy, _lib.ptr(gs), ld_gs,
                     s.data_ptr(), ld, _lib.ptr(weight), mean, mean + 4 * T, _lib.ptr(ds), _lib.ptr(dw), _lib.ptr(db), T, D)
        return ds if need[0] else None, ds if need[1] else None, dw, db, None


def _apply(what: str, x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], bias: Optional[Tensor], eps: float):
    if torch.is_autocast_enabled("cuda"):  # as F.layer_norm: in float32
        x, residual, weight, bias = (t if t is None or t.dtype not in (torch.bfloat16, torch.float16) else t.float()
                                     for t in (x, residual, weight, bias))
    index, dtype = x.get_device(), x.dtype
    if dtype not in _lib.LM_DTYPES or index < 0 or x.dim() == 0:
        raise RuntimeError(f"{what}: x must be a float32 or bfloat16 GPU tensor of at least one dimension, got {dtype} "
                           f"{tuple(x.shape)} on {x.device}")
    if residual is not None and (residual.dtype != dtype or residual.shape != x.shape or residual.get_device() != index):
        raise RuntimeError(f"{what}: residual must be as x, {dtype} {tuple(x.shape)}, got {residual.dtype} "
                           f"{tuple(residual.shape)} on {residual.device}")
    D = x.size(-1)
    kind = bias.dtype if bias is not None else dtype
    kind = weight.dtype if weight is not None and bias is None else kind
    for t in (weight, bias):
        if t is not None and (t.dtype != kind or kind != dtype and kind != torch.float32 or t.dim() != 1 or t.size(0) != D
                              or t.get_device() != index):
            raise RuntimeError(f"{what}: weight and bias must be of shape ({D},), both of x's dtype or both float32, on x's GPU, "
                               f"got {[None if t is None else (t.dtype, tuple(t.shape), str(t.device)) for t in (weight, bias)]}")
    if _lib.has_tangent((x, residual, weight, bias)):
        raise RuntimeError(f"{what} has no forward-mode derivative, and an argument carries a tangent")
    if torch.is_grad_enabled() and (x.requires_grad or residual is not None and residual.requires_grad
                                    or weight is not None and weight.requires_grad or bias is not None and bias.requires_grad):
        out = LayerNormFn.apply(x, residual, weight, bias, float(eps))
        return (out, None) if residual is None else out
    return _forward(x, residual, weight, bias, float(eps), False)[:2]


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """``F.layer_norm(x, x.shape[-1:], weight, bias, eps)`` for x [..., D], float32 or
    bfloat16 on a GPU, any strides; weight and bias [D], both of x's dtype or both float32.
    Sums and statistics are float32, the variance is about the mean; the result is rounded once.  Differentiable in
    x, weight and bias (in reverse mode; a forward-mode tangent raises), twice as torch's
    separate steps.  Under autocast it runs in float32, as ``F.layer_norm`` does."""
    return _apply("layer_norm", x, None, weight, bias, eps)[0]


def add_layer_norm(x: Tensor, residual: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                   eps: float = 1e-5) -> Tuple[Tensor, Tensor]:
    """``(layer_norm(s), s)`` with ``s = x + residual`` rounded to their dtype: the next
    block's input and residual stream.  Both outputs are differentiable."""
    return _apply("add_layer_norm", x, residual, weight, bias, eps)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension in this library's kernels; with a residual
    it returns the norm of the sum and the sum."""

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
        if x.dim() == 0 or self.normalized_shape != (x.size(-1),):
            raise RuntimeError(f"LayerNorm norms a last dimension of {tuple(self.normalized_shape)}, got {tuple(x.shape)}")
        y, s = _apply("LayerNorm", x, residual, self.weight, self.bias, self.eps)
        return y if residual is None else (y, s)


def norm_of_sum(norm: nn.Module, x: Tensor, residual: Tensor) -> Tuple[Tensor, Tensor]:
    """``(norm(s), s)`` with ``s = x + residual``: in one pass where ``norm`` is a ``LayerNorm`` and both
    are of one shape and type; a replaced or hooked one is called as it is, on torch's sum."""
    # LayerNorm sums in its terms' type, under autocast in float32
    alike = torch.promote_types(x.dtype, residual.dtype) == torch.float32 if torch.is_autocast_enabled("cuda") \
        else x.dtype == residual.dtype
    if alike and x.shape == residual.shape and calls_only(norm, LayerNorm):
        return norm.forward(x, residual)
    s = x + residual
    return norm(s), s
