"""GPU test of a stream's first call: its look-back records are clear before its kernels read
them, whatever the memory that they are allocated from held."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests.gpu_util import announce, need_gpu, no_device_errors

pytestmark = pytest.mark.gpu


def test_records_are_clear_before_the_first_kernel():
    need_gpu()
    from ossm_amd import _kernels as K

    hip = ctypes.CDLL("libamdhip64.so.7")
    gen = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=gen)  # noqa: E731
    L, B, P = 700, 1, 64
    a, g, dt = (rand(P) * 0.9 + 0.1 for _ in range(3))
    bu = torch.view_as_complex(torch.randn(L, B, P, 2, device="cuda", generator=gen))
    want = K.dlinoss_imex1_forward(a, g, dt, bu)
    torch.cuda.synchronize()
    # freed memory full of records that a stream's first launches would take for their own:
    # the first tags that the host gives, over NaN
    n = (1 << 20) + 256
    for i in range(12):
        dirt = []
        for tag in range(1, 9):
            p = ctypes.c_void_p()
            assert hip.hipMalloc(ctypes.byref(p), ctypes.c_size_t(n)) == 0
            word = (0x80000000 | tag) << 32 | 0x7fc00000
            host = (ctypes.c_uint64 * (n // 8))(*([word] * (n // 8)))
            assert hip.hipMemcpy(p, host, ctypes.c_size_t(n // 8 * 8), 1) == 0
            dirt.append(p)
        for p in dirt:
            assert hip.hipFree(p) == 0
        handle = ctypes.c_void_p()
        assert hip.hipStreamCreateWithFlags(ctypes.byref(handle), 1) == 0  # does not wait for the null stream
        announce(f"first call on fresh stream {i}")
        # work that anything on the null stream has to wait for
        busy = torch.randn(1 << 26, device="cuda").exp_().log_()
        with torch.cuda.stream(torch.cuda.ExternalStream(handle.value)):
            for k in range(3):
                got = K.dlinoss_imex1_forward(a, g, dt, bu)
                torch.cuda.synchronize()
                # look-back order varies: equal to rounding
                assert torch.isfinite(got).all() and (got - want).abs().max() <= 1e-4 * want.abs().max(), (i, k)
            no_device_errors()
        del busy
