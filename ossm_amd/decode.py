"""Serving the Mamba mixer: ragged prompts and single tokens, with states in a pool.

``mixer_prompt`` and ``mixer_step`` are the mixer between its in and out projections
(``xz`` [rows, 2 Di] to ``y`` [rows, Di], what ``MambaMixer`` trains with
``MixerCoreFn``): the causal depthwise conv + SiLU, ``x_proj``, ``dt_proj`` with its
softplus, the selective scan, the skip and the gate, in this library's kernels
(``ossm_mixer_prompt``, ``ossm_mixer_step``).

A sequence's state is what the conv and the scan remember of it: its last ``K - 1``
inputs, ``conv_state[slot]`` [K - 1, Di] (oldest first, in ``xz``'s dtype), and
``ssm_state[slot]`` [N, Di] (float32).  ``MixerState`` allocates both; the slots
are the caller's to hand out.  A slot of -1 (any index outside the pool) starts a
sequence from zeros, or keeps nothing.

xz, conv and projection weights are float32 or bfloat16, all of one dtype; dt_bias,
A_log and the skip are float32.  Sums and states are float32 and each output is
rounded once.  Inference only: a call that would need a gradient or carries a
forward-mode tangent raises.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor, nn

from . import _lib

__all__ = ["MixerState", "mixer_prompt", "mixer_step", "prompt", "step"]


class MixerState:
    """The states of ``slots`` sequences of one mixer, all zero (a new sequence's)."""

    def __init__(self, slots: int, d_inner: int, d_state: int, d_conv: int, *, dtype: torch.dtype = torch.float32,
                 device: torch.device | str = "cuda") -> None:
        self.conv = torch.zeros(slots, d_conv - 1, d_inner, dtype=dtype, device=device)
        self.ssm = torch.zeros(slots, d_state, d_inner, dtype=torch.float32, device=device)

    @classmethod
    def of(cls, mixer, slots: int, dtype: Optional[torch.dtype] = None) -> "MixerState":
        """A pool for ``mixer`` (a ``MambaMixer``), on its device."""
        w = mixer.in_proj.weight
        return cls(slots, mixer.d_inner, mixer.d_state, mixer.d_conv, dtype=dtype or w.dtype, device=w.device)


def _index(t: Optional[Tensor], n: int, name: str, what: str, dev: int) -> Optional[Tensor]:
    """An index tensor as contiguous int32 on the call's device."""
    if t is None:
        return None
    if t.dim() != 1 or t.size(0) != n or t.get_device() != dev:
        raise RuntimeError(f"{what}: {name} must be a 1-D tensor of {n} on xz's GPU, got {tuple(t.shape)} on {t.device}")
    if t.dtype != torch.int32:
        if t.dtype != torch.int64:
            raise RuntimeError(f"{what}: {name} must be int32 or int64, got {t.dtype}")
        # an index past int32 would wrap into the pool
        t = t.clamp(-1, 2**31 - 1).to(torch.int32)
    return t.contiguous()


def _args(what: str, xz: Tensor, conv_weight: Tensor, conv_bias: Optional[Tensor], x_proj: Tensor, dt_proj: Tensor,
          dt_bias: Tensor, A_log: Tensor, skip: Optional[Tensor], conv_state: Tensor, ssm_state: Tensor):
    """The checked arguments both calls share: (tensors to keep alive, dtype, sizes)."""
    dtype, dev = xz.dtype, xz.get_device()
    if dtype not in _lib.LM_DTYPES or dev < 0:
        raise RuntimeError(f"{what}: xz must be a float32 or bfloat16 GPU tensor (got {dtype} on {xz.device})")
    if xz.dim() != 2 or dt_proj.dim() != 2 or A_log.dim() != 2 or conv_weight.dim() < 2:
        raise RuntimeError(f"{what}: xz must be (rows, 2 d_inner), the weights as the mixer's, got xz {tuple(xz.shape)} "
                           f"conv weight {tuple(conv_weight.shape)} dt_proj {tuple(dt_proj.shape)} A_log {tuple(A_log.shape)}")
    Di, R = dt_proj.shape
    N, K = A_log.size(1), conv_weight.size(-1)
    slots = ssm_state.size(0)
    if xz.size(1) != 2 * Di or conv_weight.numel() != Di * K or conv_weight.size(0) != Di or \
            (conv_bias is not None and conv_bias.shape != (Di,)) or x_proj.shape != (R + 2 * N, Di) or \
            dt_bias.shape != (Di,) or A_log.shape != (Di, N) or (skip is not None and skip.shape != (Di,)) or \
            ssm_state.shape != (slots, N, Di) or conv_state.shape != (slots, K - 1, Di):
        shapes = [t if t is None else tuple(t.shape) for t in (xz, conv_weight, conv_bias, x_proj, dt_proj, dt_bias,
                                                               A_log, skip, conv_state, ssm_state)]
        raise RuntimeError(f"{what}: inconsistent shapes xz, conv weight, conv bias, x_proj, dt_proj, dt_bias, A_log, "
                           f"skip, conv_state, ssm_state: {shapes}")
    like = (conv_weight, conv_bias, x_proj, dt_proj, conv_state)
    full = (dt_bias, A_log, skip, ssm_state)
    for ts, dt in ((like, dtype), (full, torch.float32)):
        for t in ts:
            if t is not None and (t.dtype is not dt or t.get_device() != dev):
                raise RuntimeError(f"{what}: conv weight, conv bias, x_proj, dt_proj and conv_state must be {dtype}, dt_bias, "
                                   "A_log, skip and ssm_state float32, all on xz's GPU "
                                   f"(got a {t.dtype} tensor of shape {tuple(t.shape)} on {t.device})")
    if not (ssm_state.is_contiguous() and conv_state.is_contiguous()):
        raise RuntimeError(f"{what}: the state pools are updated in place and must be contiguous")
    given = (xz, *like, *full)
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in given)) or _lib.has_tangent(given):
        raise RuntimeError(f"{what} is for inference: call it under torch.no_grad() and on tensors without tangents "
                           "(MambaMixer.forward trains)")
    if xz.stride(1) != 1 or xz.stride(0) < 2 * Di:
        xz = xz.contiguous()
    weights = [t if t is None else t.contiguous() for t in (conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A_log, skip)]
    return xz, weights, (slots, Di, N, R, K)


def mixer_step(xz: Tensor, conv_weight: Tensor, conv_bias: Optional[Tensor], x_proj: Tensor, dt_proj: Tensor,
               dt_bias: Tensor, A_log: Tensor, conv_state: Tensor, ssm_state: Tensor, slots: Tensor, *,
               skip: Optional[Tensor] = None, out_slots: Optional[Tensor] = None) -> Tensor:
    """The next token of ``rows`` sequences: xz [rows, 2 Di] to y [rows, Di], row i
    continuing from ``slots[i]`` and leaving its state in ``out_slots[i]`` (default:
    the same slot).  A row whose slots are both outside the pool is padding: its y is
    zero.  No out slot may appear twice, or be another row's slot (nothing checks
    this).  Two launches, no synchronisation; it may be captured in a HIP graph
    after one eager call on the stream."""
    xz, w, (n_slots, Di, N, R, K) = _args("mixer_step", xz, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A_log,
                                          skip, conv_state, ssm_state)
    rows, dev = xz.size(0), xz.get_device()
    slots = _index(slots, rows, "slots", "mixer_step", dev)
    out_slots = _index(out_slots, rows, "out_slots", "mixer_step", dev)
    y = torch.empty((rows, Di), dtype=xz.dtype, device=xz.device)
    _lib.run(_lib.load().ossm_mixer_step, xz, _lib.LM_DTYPES[xz.dtype], xz.data_ptr(), xz.stride(0), w[0].data_ptr(),
             _lib.ptr(w[1]), w[2].data_ptr(), w[3].data_ptr(), w[4].data_ptr(), w[5].data_ptr(), _lib.ptr(w[6]),
             conv_state.data_ptr(), ssm_state.data_ptr(), slots.data_ptr(), _lib.ptr(out_slots), y.data_ptr(), rows,
             n_slots, Di, N, R, K)
    return y


def mixer_prompt(xz: Tensor, conv_weight: Tensor, conv_bias: Optional[Tensor], x_proj: Tensor, dt_proj: Tensor,
                 dt_bias: Tensor, A_log: Tensor, conv_state: Tensor, ssm_state: Tensor, slots: Tensor,
                 offsets: Tensor, resume: Optional[Tensor] = None, *, skip: Optional[Tensor] = None,
                 out_slots: Optional[Tensor] = None) -> Tensor:
    """Packed prompts: xz [rows, 2 Di] to y [rows, Di], prompt i the rows
    ``offsets[i] .. offsets[i + 1] - 1`` (offsets [prompts + 1] on the device, not
    decreasing; rows outside them are padding, y zero there).  A prompt starts from
    zeros, or from ``slots[i]`` where ``resume[i]`` (bool) is set (a prompt in pieces),
    and leaves its state in ``out_slots[i]`` (default ``slots[i]``).  Lengths may be
    anything from zero on; the host never reads them."""
    what = "mixer_prompt"
    xz, w, (n_slots, Di, N, R, K) = _args(what, xz, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A_log, skip,
                                          conv_state, ssm_state)
    rows, dev, n = xz.size(0), xz.get_device(), slots.size(0) if slots.dim() == 1 else -1
    slots = _index(slots, n, "slots", what, dev)
    out_slots = _index(out_slots, n, "out_slots", what, dev)
    offsets = _index(offsets, n + 1, "offsets", what, dev)
    if resume is not None:
        if resume.dtype not in (torch.bool, torch.uint8) or resume.shape != (n,) or resume.get_device() != dev:
            raise RuntimeError(f"{what}: resume must be a bool tensor of {n} on xz's GPU, got {resume.dtype} "
                               f"{tuple(resume.shape)} on {resume.device}")
        resume = resume.contiguous()
    y = torch.empty((rows, Di), dtype=xz.dtype, device=xz.device)
    _lib.run(_lib.load().ossm_mixer_prompt, xz, _lib.LM_DTYPES[xz.dtype], xz.data_ptr(), xz.stride(0), w[0].data_ptr(),
             _lib.ptr(w[1]), w[2].data_ptr(), w[3].data_ptr(), w[4].data_ptr(), w[5].data_ptr(), _lib.ptr(w[6]),
             conv_state.data_ptr(), ssm_state.data_ptr(), slots.data_ptr(), _lib.ptr(out_slots), offsets.data_ptr(),
             _lib.ptr(resume), y.data_ptr(), rows, n, n_slots, Di, N, R, K)
    return y


# ------------------------------------------------------------------ the module's calls
def _weights(mixer, dtype: torch.dtype):
    """A ``MambaMixer``'s parameters as the functions take them."""
    x_proj, bias = mixer.x_proj, mixer.conv1d.bias
    # the kernels take its weight alone; MambaMixer.forward calls one that does more
    if not isinstance(x_proj, nn.Linear) or type(x_proj).forward is not nn.Linear.forward or "forward" in x_proj.__dict__ \
            or x_proj.bias is not None or x_proj._forward_hooks or x_proj._forward_pre_hooks:
        raise RuntimeError("decode needs a mixer whose x_proj is an nn.Linear without bias, hooks or a forward of its own, "
                           f"got {x_proj}")
    like = [mixer.conv1d.weight.to(dtype), None if bias is None else bias.to(dtype), x_proj.weight.to(dtype),
            mixer.dt_proj.weight.to(dtype)]
    return (*like, mixer.dt_proj.bias.float(), mixer.A_log.float())


@torch.no_grad()
def prompt(mixer, inputs: Tensor, state: MixerState, slots: Tensor, offsets: Tensor,
           resume: Optional[Tensor] = None) -> Tensor:
    """``mixer`` (a ``MambaMixer``) over packed prompts, inputs [rows, d_model]; states and
    offsets as ``mixer_prompt``'s.  As in ``MambaMixer.forward`` there is no skip."""
    xz = mixer.in_proj(inputs)
    return mixer.out_proj(mixer_prompt(xz, *_weights(mixer, xz.dtype), state.conv, state.ssm, slots, offsets, resume))


@torch.no_grad()
def step(mixer, inputs: Tensor, state: MixerState, slots: Tensor) -> Tensor:
    """``mixer`` (a ``MambaMixer``) on the next token of each sequence, inputs [rows, d_model]."""
    xz = mixer.in_proj(inputs)
    return mixer.out_proj(mixer_step(xz, *_weights(mixer, xz.dtype), state.conv, state.ssm, slots))
