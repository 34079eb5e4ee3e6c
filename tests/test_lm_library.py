"""CPU-side checks of the language-model operators' boundary: the library exports
what include/ossm_lm.h declares with a ctypes signature for each, the entry points
check their arguments before any HIP call, and the Python functions refuse host
tensors.  No compute call is made."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from ossm_amd import _lib

HEADER = Path(__file__).resolve().parents[1] / "include" / "ossm_lm.h"

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libossm_scan.so not built (python -m ossm_amd.build)")


def _declarations():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return dict(re.findall(r"\b(ossm_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", text))


def test_every_declared_symbol_has_its_signature():
    found = _declarations()
    assert set(found) == set(_lib.LM_EXPORTED)
    lib = ctypes.CDLL(str(_lib.LIB_PATH))
    kinds = {"int": ctypes.c_int, "int64_t": ctypes.c_int64, "float": ctypes.c_float}
    for name, args in found.items():
        assert hasattr(lib, name), name
        want = []
        for a in [] if args.strip() in ("", "void") else args.split(","):
            pointer = "*" in a or "ossm_stream_t" in a
            want.append(ctypes.c_void_p if pointer else kinds[a.replace("const", "").split()[0]])
        assert _lib._LM_SIGNATURES[name][1] == want, name
    assert _lib.load().ossm_lm_abi_version() == 1


def _call(name, **values):
    """The entry point with pointers that are never followed and sizes of one."""
    lib, args = _lib.load(), []
    for a in _declarations()[name].split(","):
        n = a.replace("*", " ").split()[-1]
        zero = n in ("dtype", "stream")
        args.append(values.get(n, (None if n == "stream" else 0) if zero else ctypes.c_void_p(256) if "*" in a else 1))
    return getattr(lib, name)(*args), lib.ossm_last_error().decode()


@pytest.mark.parametrize("name", ["ossm_mixer_step", "ossm_mixer_prompt"])
def test_mixer_entry_points_check_before_any_hip_call(name):
    assert _call(name, dtype=7) == (1, f"{name[5:]}: unknown dtype")
    assert _call(name, rows=-1)[0] == 1 and _call(name, d_state=0)[0] == 1
    assert _call(name, d_conv=9)[0] == 3 and _call(name, d_conv=0)[0] == 3
    assert _call(name, rows=2, d_inner=4, ld_xz=7)[0] == 1
    assert _call(name, d_inner=2**21, ld_xz=2**22)[0] == 3 and _call(name, dt_rank=4000)[0] == 3
    for p in ("xz", "conv_w", "x_proj", "dt_proj", "dt_bias", "a_log", "in_slots", "y", "ssm_state"):
        assert _call(name, **{p: None}) == (1, f"{name[5:]}: null pointer")
    assert _call(name, rows=0, n_seqs=0) == (0, "")


def test_prompt_rows_need_a_sequence():
    assert _call("ossm_mixer_prompt", n_seqs=0)[0] == 1


def test_logits_entry_point_checks_before_any_hip_call():
    name = "ossm_control_logits"
    assert _call(name, dtype=2)[0] == 1 and _call(name, rows=-1)[0] == 1 and _call(name, n_bias=-1)[0] == 1
    assert _call(name, vocab=2**31)[0] == 3 and _call(name, rows=2, vocab=8, ld_out=4)[0] == 1
    for p in ("logits", "out", "history", "bias_ids", "bias_values"):
        assert _call(name, **{p: None}) == (1, "control_logits: null pointer")
    assert _call(name, rows=2**20, vocab=2**29, ld_out=2**29)[0] == 3
    assert _call(name, rows=0) == (0, "")


def test_host_tensors_are_refused():
    from ossm_amd.decode import mixer_prompt, mixer_step
    from ossm_amd.logits import control_logits

    z = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        mixer_step(z, z, None, z, z, z, z, z, z, z)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        mixer_prompt(z, z, None, z, z, z, z, z, z, z, z)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        control_logits(z)


def test_pack_allowed():
    from ossm_amd.logits import pack_allowed

    gen = torch.Generator().manual_seed(0)
    for V in (1, 31, 32, 33, 100):
        m = torch.rand(3, V, generator=gen) < 0.5
        w = pack_allowed(m)
        assert w.dtype == torch.int32 and w.shape == (3, (V + 31) // 32)
        for i in range(3):
            assert [(int(w[i, v // 32]) >> (v % 32)) & 1 for v in range(V)] == m[i].int().tolist()


@pytest.mark.parametrize("name", ["ossm_gated_forward", "ossm_gated_backward"])
def test_gated_entry_points_check_before_any_hip_call(name):
    ld = {"ld_x": 8, "ld_gate": 8, "ld_up": 8, "ld_grad": 8}
    assert _call(name, dtype=9) == (1, f"{name[5:]}: unknown dtype")
    assert _call(name, activation=5)[0] == 1 and _call(name, activation=-1)[0] == 1
    assert _call(name, rows=-1)[0] == 1 and _call(name, d_in=2)[0] == 1
    assert _call(name, ld_x=2**21)[0] == 3 and _call(name, **ld, d_out=2**20)[0] == 3
    for p in ("x", "w_gate", "w_up", "b" if name.endswith("forward") else "a"):
        assert _call(name, **ld, **{p: None}) == (1, f"{name[5:]}: null pointer")
    if name.endswith("backward"):
        assert _call(name, ld_grad=0)[0] == 1


def test_gated_refuses_host_tensors_and_unknown_activations():
    from ossm_amd.gated import GatedFeedForward, gated_linear

    z = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="one dtype on one GPU"):
        gated_linear(z, z, z)
    with pytest.raises(ValueError, match="activation"):
        gated_linear(z, z, z, activation="tanh")
    with pytest.raises(ValueError, match="activation"):
        GatedFeedForward(8, 8, activation="tanh")


def test_launches_past_32_bits_of_threads_are_refused_before_any_hip_call():
    assert _call("ossm_control_logits", rows=2**24, vocab=1) == (3, "control_logits: size exceeds launch limits")
    assert _call("ossm_control_logits", rows=2**62, vocab=1) == (3, "control_logits: size exceeds launch limits")
    big = {"d_inner": 2**17, "ld_xz": 2**18}
    assert _call("ossm_mixer_prompt", rows=2**24, ld_xz=2, dt_rank=240, d_state=64)[0] == 3  # x_proj's sums
    assert _call("ossm_mixer_prompt", rows=2**16, n_seqs=2**15, **big) == (3, "mixer_prompt: size exceeds launch limits")
