"""The gated linear recurrence: a mixer with one state a channel, whose decay each step's
input chooses.

Per channel, with a decay's parameter, an input gate i_t and a decay gate r_t (both before their
sigmoids)::

    a_t = exp(-scale * softplus(decay) * sigmoid(r_t))
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) * sigmoid(i_t) * x_t
    y_t = h_t, or h_t * silu(z_t) with an output gate z

It stands beside the scans of constant decays (``bridge.try_run_lru_scan``, the LinOSS
layers) and the selective scan of the Mamba mixer, in the forms the mixer has:
``gated_recurrence`` trains on [B, L, D] (``ossm_recurrence_forward``, ``_backward``),
``recurrence_prompt`` and ``recurrence_step`` serve packed ragged prompts and single tokens
with states in a pool (``ossm_recurrence_prompt``, ``_step``), and ``RecurrentMixer`` is
the block around them.

x and the gates are float32 or bfloat16, all of one dtype; decay and states are float32.
States and sums are float32 throughout, each output is rounded once, and results are
bitwise repeatable.  a_t is no less than 2^-126: of a state of 1e33 a step leaves 1e-5 at least.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from . import _lib
from .decode import _index
from .linear import aliases, linear

__all__ = ["GatedRecurrenceFn", "RecurrentMixer", "RecurrentState", "gated_recurrence", "recurrence_prompt",
           "recurrence_step"]


def _separate(x: Tensor, i: Tensor, r: Tensor, z: Optional[Tensor], decay: Tensor, start: Optional[Tensor],
              scale: float) -> Tuple[Tensor, Tensor]:
    """The recurrence as torch's separate steps, the scan by doubling its span."""
    l = -scale * F.softplus(decay) * torch.sigmoid(r.float())
    a = torch.exp(l)
    some = l < 0  # the root's slope at zero is infinite
    m = torch.where(some, torch.sqrt(torch.where(some, -torch.expm1(2 * l), 1.0)), 0.0)
    h = m * torch.sigmoid(i.float()) * x.float()
    if start is not None:
        h = torch.cat([h[:, :1] + a[:, :1] * start[:, None], h[:, 1:]], 1)
    span = 1
    while span < h.size(1):
        h = torch.cat([h[:, :span], h[:, span:] + a[:, span:] * h[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    y = h if z is None else h * F.silu(z.float())
    return y.to(x.dtype), h[:, -1]


def _flat(t: Tensor) -> Tuple[Tensor, int]:
    """``t`` [..., rows, D] as it is where one row stride reaches all its rows, else a
    dense copy; and that stride."""
    D = t.size(-1)
    if t.numel() == 0:
        return t, D
    ld, ok = D, t.stride(-1) == 1 or D == 1
    sizes = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n > 1]
    if sizes:
        ld = sizes[-1][1]
        ok = ok and ld >= D and (len(sizes) == 1 or sizes[0][1] == sizes[1][0] * ld)
    return (t, ld) if ok else (t.contiguous(), D)


def _pairs(*ts: Optional[Tensor]):
    """(tensors to keep alive, the pointers and row strides of each in turn)."""
    flat = [(None, 0) if t is None else _flat(t) for t in ts]
    return [t for t, _ in flat], [v for t, ld in flat for v in (_lib.ptr(t), ld)]


def _forward(x, i, r, z, decay, start, scale: float, save: bool):
    B, L, D = x.shape
    lib = _lib.load()
    keep, args = _pairs(x, i, r, z)
    decay, start = decay.contiguous(), None if start is None else start.contiguous()
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    last = torch.empty((B, D), dtype=torch.float32, device=x.device)
    saved = torch.empty(lib.ossm_recurrence_saved(B, L, D), dtype=torch.float32, device=x.device) if save else None
    if y.numel() > 0:
        _lib.run(lib.ossm_recurrence_forward, x, _lib.LM_DTYPES[x.dtype], *args, decay.data_ptr(), scale, _lib.ptr(start),
                 y.data_ptr(), last.data_ptr(), _lib.ptr(saved), B, L, D)
    return y, last, saved


def _backward(x, i, r, z, decay, gy, glast, saved, grads, scale: float, need_decay: bool, need_start: bool):
    """Gradients of x, i, r and (where there is one) z into ``grads``, tensors of one row
    stride; returns those of decay and start."""
    B, L, D = x.shape
    keep, args = _pairs(x, i, r, z)
    (gy,), gargs = _pairs(gy)
    decay = decay.contiguous()
    if glast is not None:
        glast = glast.contiguous()
    gdecay = torch.empty(D, dtype=torch.float32, device=x.device) if need_decay else None
    gstart = torch.empty((B, D), dtype=torch.float32, device=x.device) if need_start else None
    _, ld = _flat(grads[0])  # a dimension of one may have any stride
    _lib.run(_lib.load().ossm_recurrence_backward, x, _lib.LM_DTYPES[x.dtype], *gargs, _lib.ptr(glast), *args,
             decay.data_ptr(), scale, saved.data_ptr(), *(_lib.ptr(g) for g in grads), ld, _lib.ptr(gdecay), _lib.ptr(gstart),
             B, L, D)
    return gdecay, gstart


class GatedRecurrenceFn(torch.autograd.Function):
    """``gated_recurrence``; saves the state before every 32nd step."""

    @staticmethod
    def forward(ctx, x, i, r, z, decay, start, scale):  # type: ignore[override]
        y, last, saved = _forward(x, i, r, z, decay, start, scale, True)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, i, r, z, decay, start, saved)
        return y, last

    @staticmethod
    def backward(ctx, gy, glast):  # type: ignore[override]
        x, i, r, z, decay, start, saved = ctx.saved_tensors
        need = ctx.needs_input_grad
        if torch.is_grad_enabled():
            # create_graph: differentiable again, as separate steps
            inputs = aliases(x, i, r, z, decay, start)
            wanted = [t for t, n in zip(inputs, need) if n]
            outs = [(o, g) for o, g in zip(_separate(*inputs, ctx.scale), (gy, glast)) if g is not None]
            got = iter(torch.autograd.grad([o for o, _ in outs], wanted, [g for _, g in outs], create_graph=True,
                                           allow_unused=True))
            return (*(next(got) if n else None for n in need[:6]), None)
        if gy is None:
            gy = torch.zeros_like(x)
        grads = [None if t is None else torch.empty_like(x, memory_format=torch.contiguous_format) for t in (x, i, r, z)]
        gdecay, gstart = _backward(x, i, r, z, decay, gy, glast, saved, grads, ctx.scale, need[4], need[5])
        return (*(g if n else None for g, n in zip(grads, need)), gdecay, gstart, None)


class PackedRecurrenceFn(torch.autograd.Function):
    """The recurrence on the quarters x, i, r, z of one projection [B, L, 4 D]; its
    gradient is written as one tensor."""

    @staticmethod
    def forward(ctx, packed, decay, scale):  # type: ignore[override]
        packed = packed.contiguous()
        y, last, saved = _forward(*packed.chunk(4, -1), decay, None, scale, True)
        ctx.scale = scale
        ctx.save_for_backward(packed, decay, saved)
        return y

    @staticmethod
    def backward(ctx, gy):  # type: ignore[override]
        packed, decay, saved = ctx.saved_tensors
        if torch.is_grad_enabled():
            inputs = aliases(packed, decay)
            wanted = [t for t, n in zip(inputs, ctx.needs_input_grad) if n]
            y = _separate(*inputs[0].chunk(4, -1), inputs[1], None, ctx.scale)[0]
            got = iter(torch.autograd.grad(y, wanted, gy, create_graph=True))
            return (*(next(got) if n else None for n in ctx.needs_input_grad[:2]), None)
        need_p, need_d = ctx.needs_input_grad[:2]
        grad = torch.empty_like(packed)
        gdecay, _ = _backward(*packed.chunk(4, -1), decay, gy, None, saved, grad.chunk(4, -1), ctx.scale, need_d, False)
        return grad if need_p else None, gdecay, None


def _check(what: str, x: Tensor, i: Tensor, r: Tensor, z: Optional[Tensor], decay: Tensor, dims: int) -> None:
    like = (x, i, r, z)
    index = x.get_device()
    for t in like:
        if t is not None and (t.dtype != x.dtype or t.dtype not in _lib.LM_DTYPES or index < 0 or t.get_device() != index):
            raise RuntimeError(f"{what}: x and the gates must be float32 or bfloat16 tensors of one dtype on one GPU, got "
                               f"{[None if t is None else (t.dtype, str(t.device)) for t in like]}")
    if x.dim() != dims or any(t is not None and t.shape != x.shape for t in like):
        raise RuntimeError(f"{what}: x and the gates must be {'(batch, length, channels)' if dims == 3 else '(rows, channels)'}, "
                           f"all of one shape, got {[None if t is None else tuple(t.shape) for t in like]}")
    if decay.dtype != torch.float32 or decay.shape != x.shape[-1:] or decay.get_device() != index:
        raise RuntimeError(f"{what}: decay must be a float32 tensor ({x.size(-1)},) on x's GPU, got {decay.dtype} "
                           f"{tuple(decay.shape)} on {decay.device}")


def gated_recurrence(x: Tensor, input_gate: Tensor, decay_gate: Tensor, decay: Tensor, output_gate: Optional[Tensor] = None,
                     state: Optional[Tensor] = None, *, scale: float = 8.0) -> Tuple[Tensor, Tensor]:
    """(y [B, L, D], the states after the last step [B, D]) of the recurrence over x
    [B, L, D] and its gates (of x's dtype and shape, any strides) with decay float32 [D], from
    state float32 [B, D] (default zeros); scale is positive and finite.  Differentiable in every tensor (in reverse mode; a
    forward-mode tangent raises), twice as torch's separate steps."""
    what = "gated_recurrence"
    _check(what, x, input_gate, decay_gate, output_gate, decay, 3)
    B, L, D = x.shape
    if state is not None and (state.dtype != torch.float32 or state.shape != (B, D) or state.get_device() != x.get_device()):
        raise RuntimeError(f"{what}: state must be a float32 tensor ({B}, {D}) on x's GPU, got {state.dtype} "
                           f"{tuple(state.shape)} on {state.device}")
    args = (x, input_gate, decay_gate, output_gate, decay, state)
    if _lib.has_tangent(args):
        raise RuntimeError(f"{what} has no forward-mode derivative, and an argument carries a tangent")
    if L == 0 or B == 0 or D == 0:  # nothing happens to the states
        last = x.new_zeros((B, D), dtype=torch.float32) if state is None else state.clone()
        return x * 0.0, last
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        return GatedRecurrenceFn.apply(*args, float(scale))
    return _forward(*args, float(scale), False)[:2]


def _serve(what: str, x: Tensor, i: Tensor, r: Tensor, z: Optional[Tensor], decay: Tensor, state: Tensor) -> None:
    _check(what, x, i, r, z, decay, 2)
    if state.dtype != torch.float32 or state.dim() != 2 or state.size(1) != x.size(1) or state.get_device() != x.get_device() \
            or not state.is_contiguous():
        raise RuntimeError(f"{what}: state is updated in place and must be a contiguous float32 tensor (slots, {x.size(1)}) on "
                           f"x's GPU, got {state.dtype} {tuple(state.shape)} strides {state.stride()} on {state.device}")
    given = (x, i, r, z, decay, state)
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in given)) or _lib.has_tangent(given):
        raise RuntimeError(f"{what} is for inference: call it under torch.no_grad() and on tensors without tangents "
                           "(gated_recurrence trains)")


def recurrence_prompt(x: Tensor, input_gate: Tensor, decay_gate: Tensor, decay: Tensor, state: Tensor, slots: Tensor,
                      offsets: Tensor, resume: Optional[Tensor] = None, *, output_gate: Optional[Tensor] = None,
                      scale: float = 8.0, out_slots: Optional[Tensor] = None) -> Tensor:
    """Packed prompts: x and the gates [rows, D] to y [rows, D], prompt i the rows
    ``offsets[i] .. offsets[i + 1] - 1``, states in the pool ``state`` [slots, D];
    slots, offsets, resume, out_slots and padding as ``decode.mixer_prompt``'s.  The host
    never reads the lengths."""
    what = "recurrence_prompt"
    _serve(what, x, input_gate, decay_gate, output_gate, decay, state)
    (rows, D), dev, n = x.shape, x.get_device(), slots.size(0) if slots.dim() == 1 else -1
    slots, out_slots = _index(slots, n, "slots", what, dev), _index(out_slots, n, "out_slots", what, dev)
    offsets = _index(offsets, n + 1, "offsets", what, dev)
    if resume is not None:
        if resume.dtype not in (torch.bool, torch.uint8) or resume.shape != (n,) or resume.get_device() != dev:
            raise RuntimeError(f"{what}: resume must be a bool tensor of {n} on x's GPU, got {resume.dtype} "
                               f"{tuple(resume.shape)} on {resume.device}")
        resume = resume.contiguous()
    keep, args = _pairs(x, input_gate, decay_gate, output_gate)
    decay = decay.contiguous()
    y = torch.empty((rows, D), dtype=x.dtype, device=x.device)
    _lib.run(_lib.load().ossm_recurrence_prompt, x, _lib.LM_DTYPES[x.dtype], *args, decay.data_ptr(), scale, state.data_ptr(),
             slots.data_ptr(), _lib.ptr(out_slots), offsets.data_ptr(), _lib.ptr(resume), y.data_ptr(), rows, n,
             state.size(0), D)
    return y


def recurrence_step(x: Tensor, input_gate: Tensor, decay_gate: Tensor, decay: Tensor, state: Tensor, slots: Tensor, *,
                    output_gate: Optional[Tensor] = None, scale: float = 8.0, out_slots: Optional[Tensor] = None) -> Tensor:
    """The next token of ``rows`` sequences: x and the gates [rows, D] to y [rows, D], row i
    continuing from ``state[slots[i]]`` and leaving its state in ``out_slots[i]`` (default the same
    slot), both as ``decode.mixer_step``'s.  One launch, no synchronisation, no workspace."""
    what = "recurrence_step"
    _serve(what, x, input_gate, decay_gate, output_gate, decay, state)
    rows, D = x.shape
    dev = x.get_device()
    slots, out_slots = _index(slots, rows, "slots", what, dev), _index(out_slots, rows, "out_slots", what, dev)
    keep, args = _pairs(x, input_gate, decay_gate, output_gate)
    decay = decay.contiguous()
    y = torch.empty((rows, D), dtype=x.dtype, device=x.device)
    _lib.run(_lib.load().ossm_recurrence_step, x, _lib.LM_DTYPES[x.dtype], *args, decay.data_ptr(), scale, state.data_ptr(),
             slots.data_ptr(), _lib.ptr(out_slots), y.data_ptr(), rows, state.size(0), D)
    return y


class RecurrentState:
    """The states of ``slots`` sequences of one ``RecurrentMixer``, all zero (a new
    sequence's)."""

    def __init__(self, slots: int, d_inner: int, *, device: torch.device | str = "cuda") -> None:
        self.h = torch.zeros(slots, d_inner, dtype=torch.float32, device=device)

    @classmethod
    def of(cls, mixer: "RecurrentMixer", slots: int) -> "RecurrentState":
        """A pool for ``mixer``, on its device."""
        return cls(slots, mixer.d_inner, device=mixer.in_proj.weight.device)


class RecurrentMixer(nn.Module):
    """A block's mixer on the gated linear recurrence: one projection to x and its three
    gates, the recurrence, one projection back.  ``forward`` trains on [B, L, d_model];
    ``prompt`` and ``step`` serve, as ``decode.prompt`` and ``decode.step`` serve a ``MambaMixer``."""

    def __init__(self, d_model: int, *, expand: int = 2, scale: float = 8.0, bias: bool = False) -> None:
        super().__init__()
        if not 0.0 < scale < math.inf:
            raise ValueError(f"scale must be positive and finite, not {scale!r}")
        self.d_model, self.d_inner, self.scale = d_model, expand * d_model, scale
        self.in_proj = nn.Linear(d_model, 4 * self.d_inner, bias=bias)
        self.out_proj = nn.Linear(self.d_inner, d_model, bias=bias)
        # at a gate half open a channel remembers 10 to 1000 steps
        rate = torch.exp(torch.empty(self.d_inner).uniform_(math.log(1e-3), math.log(0.1)))
        self.decay = nn.Parameter(torch.log(torch.expm1(2 * rate / scale)))

    def forward(self, inputs: Tensor) -> Tensor:
        packed, decay = linear(self.in_proj, inputs), self.decay.float()
        if torch.is_grad_enabled() and (packed.requires_grad or decay.requires_grad) and packed.numel() > 0:
            x, i, r, z = packed.chunk(4, -1)
            _check("RecurrentMixer", x, i, r, z, decay, 3)
            if _lib.has_tangent((packed, decay)):
                raise RuntimeError("RecurrentMixer has no forward-mode derivative, and an argument carries a tangent")
            y = PackedRecurrenceFn.apply(packed, decay, float(self.scale))
        else:
            x, i, r, z = packed.chunk(4, -1)
            y = gated_recurrence(x, i, r, decay, z, scale=self.scale)[0]
        return linear(self.out_proj, y)

    @torch.no_grad()
    def prompt(self, inputs: Tensor, state: RecurrentState, slots: Tensor, offsets: Tensor,
               resume: Optional[Tensor] = None) -> Tensor:
        """Packed prompts, inputs [rows, d_model]; states and offsets as ``recurrence_prompt``'s."""
        x, i, r, z = self.in_proj(inputs).chunk(4, -1)
        return self.out_proj(recurrence_prompt(x, i, r, self.decay.float(), state.h, slots, offsets, resume, output_gate=z,
                                               scale=self.scale))

    @torch.no_grad()
    def step(self, inputs: Tensor, state: RecurrentState, slots: Tensor) -> Tensor:
        """The next token of each sequence, inputs [rows, d_model]."""
        x, i, r, z = self.in_proj(inputs).chunk(4, -1)
        return self.out_proj(recurrence_step(x, i, r, self.decay.float(), state.h, slots, output_gate=z, scale=self.scale))
