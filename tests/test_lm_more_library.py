"""CPU-side checks of layer norm's, the recurrence's and the sampler's boundary: the entry
points check their arguments before any HIP call, and the Python functions refuse host
tensors.  No compute call is made."""

from __future__ import annotations

import pytest
import torch

from ossm_amd import _lib
from tests.test_lm_library import _call, _declarations

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libossm_scan.so not built (python -m ossm_amd.build)")


@pytest.mark.parametrize("name", ["ossm_layer_norm_forward", "ossm_layer_norm_backward"])
def test_layer_norm_checks_before_any_hip_call(name):
    ok = {"weight_dtype": 0}
    assert _call(name, dtype=3, **ok) == (1, f"{name[5:]}: unknown dtype")
    assert _call(name, dtype=0, weight_dtype=1) == (1, f"{name[5:]}: unknown dtype")
    assert _call(name, dtype=1, weight_dtype=2)[0] == 1
    assert _call(name, rows=-1, **ok)[0] == 1 and _call(name, dim=-1, **ok)[0] == 1
    assert _call(name, dim=2**40, **ok)[0] == 3
    assert _call(name, rows=0, **ok) == (0, "") and _call(name, dim=0, **ok) == (0, "")
    required = ("x", "y", "mean", "sum") if name.endswith("forward") else ("grad_y", "s", "mean", "rstd")
    for p in required:
        assert _call(name, **ok, **{p: None}) == (1, f"{name[5:]}: null pointer")
    assert _call(name, rows=2, dim=8, **ok) == (1, f"{name[5:]}: row stride below the row")


@pytest.mark.parametrize("name", ["ossm_recurrence_forward", "ossm_recurrence_backward"])
def test_recurrence_training_checks_before_any_hip_call(name):
    assert _call(name, dtype=2) == (1, f"{name[5:]}: unknown dtype")
    for size in ("batch", "length", "dim"):
        assert _call(name, **{size: -1})[0] == 1 and _call(name, **{size: 2**40})[0] == 3
        assert _call(name, **{size: 0}) == (0, "")
    for p in ("x", "input_gate", "decay_gate", "decay", *(("y", "last") if name.endswith("forward") else ("grad_y", "saved", "grad_x", "grad_input_gate", "grad_decay_gate",
                                                                "grad_output_gate", "output_gate"))):
        assert _call(name, **{p: None}) == (1, f"{name[5:]}: null pointer")
    assert _call(name, length=2, dim=8) == (1, f"{name[5:]}: row stride below the row")


@pytest.mark.parametrize("name", ["ossm_recurrence_prompt", "ossm_recurrence_step"])
def test_recurrence_serving_checks_before_any_hip_call(name):
    assert _call(name, dtype=2) == (1, f"{name[5:]}: unknown dtype")
    assert _call(name, rows=-1)[0] == 1 and _call(name, n_slots=-1)[0] == 1 and _call(name, n_slots=2**31)[0] == 1
    for p in ("x", "input_gate", "decay_gate", "decay", "y", "state", "in_slots"):
        assert _call(name, **{p: None}) == (1, f"{name[5:]}: null pointer")
    assert _call(name, rows=2, dim=8) == (1, f"{name[5:]}: row stride below the row")
    assert _call(name, rows=0, n_seqs=0) == (0, "") and _call(name, dim=0) == (0, "")
    if name.endswith("prompt"):
        assert _call(name, n_seqs=65536)[0] == 3 and _call(name, n_seqs=-1)[0] == 1
        assert _call(name, offsets=None) == (1, "recurrence_prompt: null pointer")


@pytest.mark.parametrize("name", [f"ossm_recurrence_{w}" for w in ("forward", "backward", "prompt", "step")])
def test_recurrence_needs_a_positive_scale(name):
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert _call(name, scale=scale) == (1, f"{name[5:]}: scale must be positive and finite")


def test_sampler_checks_before_any_hip_call():
    name = "ossm_sample_logits"
    assert _call(name, dtype=2) == (1, "sample_logits: unknown dtype")
    assert _call(name, rows=-1)[0] == 1 and _call(name, vocab=-1)[0] == 1 and _call(name, vocab=0)[0] == 1
    assert _call(name, vocab=2**20 + 1)[0] == 3 and _call(name, rows=2**40)[0] == 3
    for p in ("logits", "uniform", "tokens"):
        assert _call(name, **{p: None}) == (1, "sample_logits: null pointer")
    assert _call(name, rows=0) == (0, "")


def test_saved_states_are_one_every_32_steps():
    lib = _lib.load()
    assert [lib.ossm_recurrence_saved(2, n, 3) for n in (1, 32, 33, 64, 65)] == [6, 6, 12, 12, 18]
    assert "ossm_recurrence_saved" in _declarations()


def test_host_tensors_are_refused():
    from ossm_amd.norm import LayerNorm, add_layer_norm, layer_norm
    from ossm_amd.recurrence import RecurrentMixer, gated_recurrence, recurrence_prompt, recurrence_step
    from ossm_amd.sampling import sample_logits

    z = torch.zeros(2, 8)
    for call in (lambda: layer_norm(z), lambda: add_layer_norm(z, z), lambda: LayerNorm(8)(z), lambda: sample_logits(z, z[:, 0])):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()
    for call in (lambda: gated_recurrence(z[None], z[None], z[None], z[0]), lambda: recurrence_step(z, z, z, z[0], z, z[:, 0]),
                 lambda: recurrence_prompt(z, z, z, z[0], z, z[:, 0], z[:, 0]), lambda: RecurrentMixer(8)(z[None])):
        with pytest.raises(RuntimeError, match="one GPU"):
            call()


def test_separate_steps_match_a_loop():
    """The composition that second derivatives go through, against a loop in float64 (it holds
    the dtype that it is given in its states)."""
    from ossm_amd.recurrence import _separate

    torch.manual_seed(0)
    x, i, r, z = (torch.randn(2, 13, 5) for _ in range(4))
    decay, start = torch.randn(5), torch.randn(2, 5)
    y, last = _separate(x, i, r, z, decay, start, 8.0)
    h = start.double()
    for t in range(13):
        a = torch.exp(-8 * torch.nn.functional.softplus(decay.double()) * torch.sigmoid(r[:, t].double()))
        h = a * h + torch.sqrt(1 - a * a) * torch.sigmoid(i[:, t].double()) * x[:, t].double()
        assert (y[:, t] - h * torch.nn.functional.silu(z[:, t].double())).abs().max() < 1e-5
    assert (last - h).abs().max() < 1e-5


def test_recurrence_gradients_stay_in_their_tensor(monkeypatch):
    """A projection of one step whose step's stride is any number (such a tensor is contiguous): every
    row of the gradients, at the row stride that the library is given, lies in the tensor."""
    from ossm_amd import recurrence

    calls = []
    monkeypatch.setattr(_lib, "run", lambda fn, t, *args: calls.append((fn.__name__, args)))
    B, D = 5, 4
    for packed in (torch.zeros(1, B, 4 * D).transpose(0, 1), torch.zeros(B, 1, 4 * D),
                   torch.zeros(4 * D * B).as_strided((B, 1, 4 * D), (4 * D, 10 ** 6, 1))):
        assert packed.is_contiguous()
        packed.requires_grad_(True)
        y = recurrence.PackedRecurrenceFn.apply(packed, torch.zeros(D), 8.0)
        grad, = torch.autograd.grad(y, packed, torch.zeros_like(y))
        assert grad.shape == packed.shape
        name, args = calls[-1]
        assert name == "ossm_recurrence_backward"
        # dtype, grad_y, its stride, grad_last, x and gates with strides, decay, scale, saved, four gradients, their stride
        assert args[4 + 8 + 3 + 4] == 4 * D


def test_only_bare_modules_are_passed_by():
    """What a caller may do in a module's place: nothing where anything else is called with it."""
    from torch import nn

    from ossm_amd.linear import calls_only
    from ossm_amd.norm import LayerNorm

    assert calls_only(LayerNorm(8), LayerNorm) and not calls_only(nn.LayerNorm(8), LayerNorm)
    none = lambda *a: None  # noqa: E731
    for change in (lambda m: m.register_forward_hook(none), lambda m: m.register_forward_pre_hook(none),
                   lambda m: m.register_full_backward_hook(none), lambda m: m.register_full_backward_pre_hook(none),
                   lambda m: setattr(m, "forward", none), lambda m: m.compile()):
        m = LayerNorm(8)
        change(m)
        assert not calls_only(m, LayerNorm)

    class Own(LayerNorm):
        def forward(self, x, residual=None):
            return x

    assert not calls_only(Own(8), LayerNorm) and calls_only(type("Same", (LayerNorm,), {})(8), LayerNorm)
    handle = nn.modules.module.register_module_forward_hook(none)
    try:
        assert not calls_only(LayerNorm(8), LayerNorm)
    finally:
        handle.remove()
