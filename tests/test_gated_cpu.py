"""CPU-side checks of ossm_amd.gated's Python: what it tells the kernels of a matrix.
No kernel runs."""

from __future__ import annotations

import pytest
import torch

from ossm_amd import gated

WIDE = (1 << 20) + 8  # past the row stride that the kernels take


def _views():
    base = torch.arange(1.0, 1 + 3 * 40).view(3, 40)
    one = torch.tensor([[3.0]])
    yield "dense", base
    yield "rows of a wider matrix", base[:, 5:12]
    yield "transposed", base.t()
    yield "one row of all", base[:1].expand(6, 40)
    yield "one element of all", one.expand(5, 1)
    yield "one element, one column of many", one.expand(5, 7)
    yield "a summed loss's gradient of one column", torch.ones(()).expand(9, 1)
    yield "one column", base[:, 3:4]
    yield "every other of one column", base[::2, 3:4]
    yield "one column of a transposed matrix", base.t()[:, 1:2]
    yield "one column of a very wide matrix", torch.empty(2, WIDE).fill_(2.0)[:, :1]
    yield "columns of a very wide matrix", torch.empty(2, WIDE).fill_(2.0)[:, :3]
    yield "one row", base[1:2, ::3]
    yield "one element", base[2:, 7:8]
    yield "no columns of a very wide matrix", torch.empty(2, WIDE)[:, :0]
    yield "no rows", base[:0]


@pytest.mark.parametrize("name", [n for n, _ in _views()])
def test_a_matrix_is_described_as_it_lies(name):
    """Rows at the stride told to the kernels are the matrix's and lie inside its storage."""
    t = dict(_views())[name]
    m = gated._matrix(t)
    rows, cols = m.shape
    assert m.shape == t.shape and cols <= gated._ld(m) <= 1 << 20
    if m.numel() == 0:
        return
    end = m.storage_offset() + (rows - 1) * gated._ld(m) + cols
    assert end <= m.untyped_storage().nbytes() // m.element_size()
    assert torch.equal(m.as_strided((rows, cols), (gated._ld(m), 1)), t)


class _OnHost:
    """GatedLinearFn with its forward as torch's steps: the backward under create_graph
    runs no kernel."""

    def __init__(self, monkeypatch):
        monkeypatch.setattr(gated, "_forward", lambda x, wg, wu, bg, bu, act, save: (
            gated._separate(x, wg, wu, bg, bu, act), *(torch.nn.functional.linear(x, *p) for p in ((wg, bg), (wu, bu)))))

    def __call__(self, *args):
        return gated.GatedLinearFn.apply(*args, "silu")


def _tied(f):
    """The gate's weight is the up weight too, as are the biases."""
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(*s, dtype=torch.float64, generator=g).requires_grad_(True) for s in ((6, 5), (4, 5), (4,)))
    return f(x, w, w, b, b), [x, w, b]


def _twice(f):
    """One block applied to its own output."""
    g = torch.Generator().manual_seed(2)
    x, wg, wu, b = (torch.randn(*s, dtype=torch.float64, generator=g).requires_grad_(True)
                    for s in ((6, 5), (5, 5), (5, 5), (5,)))
    return f(f(x, wg, wu, b, None), wg, wu, b, None), [x, wg, wu, b]


@pytest.mark.parametrize("use", [_tied, _twice])
def test_shared_inputs_differentiate_twice(monkeypatch, use):
    """Under create_graph each path to a shared tensor counts once, in the gradients and in theirs."""
    seen = []
    for f in (_OnHost(monkeypatch), lambda *a: gated._separate(*a, "silu")):
        y, leaves = use(f)
        grads = torch.autograd.grad(y.square().sum(), leaves, create_graph=True)
        seen.append((*grads, *torch.autograd.grad(sum(t.square().sum() for t in grads), leaves, create_graph=True)))
    for a, b in zip(*seen):
        assert torch.allclose(a, b, rtol=1e-10, atol=1e-10 * float(b.detach().abs().max()))
