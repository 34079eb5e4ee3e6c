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
