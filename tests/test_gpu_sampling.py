"""GPU tests of sample_logits against a row-by-row computation in extended precision:
tokens are whole numbers and have to be equal.

A weight is off by less than 2^-43 of the largest, so a running sum by 2^-43 V of the
whole at the most; of the tests' random rows (some 10^4, borders at the vocabulary's
tokens) one lands that near a border with a chance below 10^-4 in all."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(scope="module")
def S():
    need_gpu()
    from ossm_amd import sampling

    return sampling


def reference(logits, u, temperature, top_k, top_p, min_p):
    """One row, all in float64 and longdouble."""
    row = logits.astype(np.float64).copy()
    row[np.isnan(row)] = -INF
    if row.max() == -INF:
        return -1
    if not temperature > 0:
        return int(row.argmax())
    ids = np.argsort(-row, kind="stable")
    ids = ids[row[ids] > -INF]
    if top_k > 0:
        ids = ids[:top_k]
    top = row[ids[0]]
    if top == INF:
        w = (row[ids] == INF).astype(np.longdouble)
    else:
        with np.errstate(under="ignore", over="ignore"):
            w = np.exp(((row[ids] - top) / np.float64(temperature)).astype(np.longdouble))
    w[w < 2.0 ** -60] = 0
    if top_p < 1:
        cum = np.cumsum(w)
        n = 1 + int((cum[:-1] < np.longdouble(top_p) * cum[-1]).sum())
        ids, w = ids[:n], w[:n]
    if min_p > 0:
        n = max(1, int((w >= min(1.0, float(min_p))).sum()))
        ids, w = ids[:n], w[:n]
    order = np.argsort(ids)
    cum = np.cumsum(w[order])
    at = int(np.searchsorted(cum, np.longdouble(min(max(float(u), 0.0), 1.0)) * cum[-1], side="right"))
    return int(ids[order][at]) if at < len(ids) else int(ids[order][np.nonzero(w[order])[0][-1]])


def check(S, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, **kw):
    """Settings as numbers or arrays a row."""
    rows = x.size(0)
    every = lambda v, t: np.broadcast_to(np.asarray(v, t), (rows,))  # noqa: E731
    t, k, p, m = every(temperature, np.float32), every(top_k, np.int64), every(top_p, np.float32), every(min_p, np.float32)
    give = lambda v, a, t: torch.tensor(a.astype(t)).cuda() if np.ndim(v) else v  # noqa: E731
    got = S.sample_logits(x, torch.tensor(np.asarray(u, np.float32)).cuda(), temperature=give(temperature, t, np.float32),
                          top_k=give(top_k, k, np.int32), top_p=give(top_p, p, np.float32),
                          min_p=give(min_p, m, np.float32), **kw)
    assert got.dtype == torch.int64 and got.shape == (rows,)
    logits = x.double().cpu().numpy()
    want = [reference(logits[i], np.asarray(u, np.float32)[i], t[i], k[i], p[i], m[i]) for i in range(rows)]
    assert got.tolist() == want, [(i, a, b) for i, (a, b) in enumerate(zip(got.tolist(), want)) if a != b][:5]
    return got


SIZES = [(1, 1), (3, 2), (8, 31), (40, 500), (5, 511), (6, 512), (7, 513), (9, 4099), (3, 8191), (4, 8192), (5, 8193),
         (2, 50001), (33, 1003), (2, 131072), (1, 262147)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_matches_extended_precision(S, size, dtype):
    rows, V = size
    rng = np.random.default_rng(V)
    announce(f"sample_logits {size} {dtype}")
    for scale in (0.1, 1.0, 3.0, 20.0):
        x = torch.tensor(rng.normal(size=size) * scale).to(dtype).cuda()
        u = rng.random(rows)
        check(S, x, u)
        check(S, x, u, 0.7, min(V, 40))
        check(S, x, u, 0.9, 0, 0.9)
        check(S, x, u, 1.1, 0, 1.0, 0.05)
        mixed = dict(temperature=rng.choice([0.0, 0.3, 1.0, 5.0], rows), top_k=rng.integers(-1, V + 2, rows),
                     top_p=rng.choice([0.0, 0.1, 0.5, 0.97, 1.0, 2.0], rows), min_p=rng.choice([0.0, 0.001, 0.3, 1.0, 3.0], rows))
        check(S, x, u, **mixed)
        x[:, 1::3] = -INF
        check(S, x, u, **mixed)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_ties_go_to_the_lowest_index(S, dtype):
    """Equal logits: k and p keep the first of them; 0 and -0 are equal."""
    V = 3000
    u = np.arange(64) / 64
    for row in (np.zeros(V), np.where(np.arange(V) % 2, 0.0, -0.0), np.arange(V) // 700 * 1.0, np.arange(V)[::-1] // 100 * -0.5,
                np.where(np.arange(V) % 5 == 2, 1.0, 0.5)):
        x = torch.tensor(np.broadcast_to(row, (64, V)).copy()).to(dtype).cuda()
        announce("sample_logits ties")
        check(S, x, u)
        for k in (1, 2, 3, 599, 600, 601, 1500, 2999, 3000, 3001):
            check(S, x, u, 1.0, k)
        for p in (0.0, 2.0 ** -20, 0.25, 0.5, 0.75, 0.999):  # halves and quarters land on a border exactly
            check(S, x, u, 1.0, 0, p)
            check(S, x, u, 2.0, 1000, p)
    x = torch.zeros(4, 8).to(dtype).cuda()
    got = S.sample_logits(x, torch.tensor([0.0, 0.24, 0.25, 0.49]).cuda(), top_p=0.5)  # four of eight kept
    assert got.tolist() == [0, 0, 1, 1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_borders_of_p_and_min_p_next_to_each_other(S, dtype):
    announce(dtype)
    V, rng = 40000, np.random.default_rng(91)
    x = torch.tensor(rng.normal(size=(1, V)), dtype=dtype)
    w = np.sort(np.exp(x.double().numpy()[0] - float(x.max())))[::-1]
    rows = []
    for part in (0.05, 0.3, 0.7, 0.97):
        border = w[int((np.cumsum(w) < part * w.sum()).sum())]
        for near in (0.5, 0.999, 0.99999, 1.0, 1.00001, 1.001, 2.0):
            for k in (0, 900, 20000):
                rows.append((part, border * near, k))
    part, floor, k = (np.array(c) for c in zip(*rows))
    u = rng.uniform(size=len(rows))
    check(S, x.expand(len(rows), V).contiguous().cuda(), u, 1.0, k, part, floor)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_crowded_and_sparse_rows(S, dtype):
    announce(dtype)
    V, rng = 30000, np.random.default_rng(92)
    crowd = np.full(V, -9.0)
    crowd[rng.permutation(V)[:3000]] = 2.0
    crowd[[77, 29999]] = 2.015625, 2.0078125  # one bin's width of the row's, far apart in bits
    coarse = np.round(rng.normal(size=V) * 8) / 8
    masked = np.where(np.arange(V) % 8 == 1, rng.normal(size=V), -INF)  # none of every eighth is left
    deep = rng.normal(size=V)
    deep[::8] = 4.0
    deep[1::2] -= 300.0  # far below what every eighth reaches
    for row in (crowd, coarse, masked, deep):
        x = torch.tensor(np.stack([row] * 24), dtype=dtype).cuda()
        u = rng.uniform(size=24)
        part = np.array([0.02, 0.4, 0.8, 0.99] * 6)
        for kw in ({"top_p": part}, {"top_k": 600}, {"top_k": 2500}, {"top_k": 9000, "top_p": part},
                   {"top_p": part, "min_p": 0.3}, {"temperature": 7.0, "top_p": part}):
            check(S, x, u, **kw)


def test_special_values(S):
    V = 700
    rng = np.random.default_rng(0)
    base = rng.normal(size=V)
    rows = []
    for change in ({3: np.nan}, {5: INF}, {5: INF, 600: INF, 6: -INF}, {i: -INF for i in range(V)}, {i: np.nan for i in range(V)},
                   {i: -INF for i in range(V) if i != 77}, {i: float(np.finfo(np.float32).min) for i in range(0, V, 2)},
                   {0: float(np.finfo(np.float32).max)}, {i: float(np.finfo(np.float32).min) for i in range(V)},
                   {9: 1e30, 10: 1e30}, {i: -1e-42 for i in range(V)}):
        r = base.copy()
        for i, v in change.items():
            r[i] = v
        rows.append(r)
    x = torch.tensor(np.array(rows)).float().cuda()
    n = len(rows)
    announce("sample_logits special values")
    for u in (0.0, 0.3, 0.9999999):
        us = np.full(n, u)
        for t in (1.0, 0.0, -1.0, 1e-30, 1e30, INF, float("nan"), 1e-42):
            check(S, x, us, t)
            check(S, x, us, t, 3)
            check(S, x, us, t, 0, 0.6)
            check(S, x, us, t, 5, 0.6, 0.2)
    plain = x[:1].expand(4, V)
    for value in (-0.5, 1.0, 7.0):  # numbers outside [0, 1) count as the nearest inside
        got = S.sample_logits(torch.nan_to_num(plain), torch.full((4,), value).cuda())
        assert got.tolist() == ([0] * 4 if value < 0 else [V - 1] * 4)


def test_random_numbers_at_the_borders(S):
    """u on the running sum itself: the next token; the largest below one: the last."""
    x = torch.log(torch.tensor([[1.0, 2.0, 4.0, 1.0]])).cuda().expand(6, 4).contiguous()
    x = torch.zeros(6, 8).cuda()
    u = torch.tensor([0.0, 0.125, 0.25, 0.5, 0.875, 1 - 2.0 ** -24]).cuda()
    announce("sample_logits at borders")
    assert S.sample_logits(x, u).tolist() == [0, 1, 2, 4, 7, 7]
    tiny = torch.full((2, 8), 0.0).cuda()
    assert S.sample_logits(tiny, torch.tensor([1e-45, 2.0 ** -126]).cuda()).tolist() == [0, 0]


def test_strides_offsets_out_and_other_streams(S):
    rows, V = 6, 5003
    rng = np.random.default_rng(1)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.tensor(rng.normal(size=(rows, V)) * 2).to(dtype).cuda()
        u = rng.random(rows)
        want = check(S, x, u, 0.8, 100, 0.9, 0.01)
        tu = torch.tensor(u).float().cuda()
        for off in range(9):
            view = torch.zeros(rows, V + 30, dtype=dtype, device="cuda")[:, off:off + V].copy_(x)
            out = torch.full((2 * rows,), -7, dtype=torch.int64, device="cuda")
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            announce(f"sample_logits offset {off} {dtype}")
            with torch.cuda.stream(side):
                got = S.sample_logits(view, tu, temperature=0.8, top_k=100, top_p=0.9, min_p=0.01, out=out[::2])
            torch.cuda.synchronize()
            assert torch.equal(got, want) and torch.equal(out[::2], want) and torch.all(out[1::2] == -7)
        got = S.sample_logits(x.t().contiguous().t(), tu, temperature=0.8, top_k=100, top_p=0.9, min_p=0.01)
        assert torch.equal(got, want)
        one = S.sample_logits(x[:1].expand(rows, V), tu, temperature=0.8)
        assert torch.equal(one, S.sample_logits(x[:1].repeat(rows, 1), tu, temperature=0.8))
        long = S.sample_logits(x, tu, temperature=0.8, top_k=torch.full((rows,), 100).cuda(), top_p=0.9, min_p=0.01)
        assert torch.equal(long, want)


def test_logits_past_32_bits(S):
    rows, V = 11000, 200003
    assert (rows - 1) * V > 2 ** 31
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(2)
    x[-3:] = torch.tensor(rng.normal(size=(3, V)) * 3).bfloat16().cuda()
    u = rng.random(3)
    announce("sample_logits past 2^31 elements")
    want = check(S, x[-3:], u, 0.9, 0, 0.95)
    tu = torch.zeros(rows, device="cuda")
    tu[-3:] = torch.tensor(u).float().cuda()
    got = S.sample_logits(x, tu, temperature=0.9, top_p=0.95)
    assert torch.equal(got[-3:], want) and torch.all(got[:-3] == 0)


def test_the_largest_vocabulary(S):
    V = 2 ** 20
    rng = np.random.default_rng(3)
    x = torch.tensor(rng.normal(size=(2, V))).float().cuda()
    announce("sample_logits 2^20")
    for kw in ({}, {"top_k": 70000}, {"top_p": 0.7}, {"min_p": 0.1}):
        check(S, x, rng.random(2), 1.0, **kw)
        check(S, x.bfloat16(), rng.random(2), 1.0, **kw)
    with pytest.raises(RuntimeError, match="1 to 2\\^20"):
        S.sample_logits(torch.zeros(1, V + 1).cuda(), torch.zeros(1).cuda())


def test_graph_capture(S):
    rows, V = 5, 6000
    x = torch.randn(rows, V).cuda() * 3
    u, k = torch.rand(rows).cuda(), torch.tensor([0, 1, 50, 3000, 9000], dtype=torch.int32).cuda()
    p = torch.tensor([0.9, 1.0, 0.5, 0.99, 0.1]).cuda()
    call = lambda: S.sample_logits(x, u, temperature=0.9, top_k=k, top_p=p, min_p=0.001)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    announce("sample_logits under graph capture")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    for i in range(6):
        x.normal_()
        u.uniform_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, call()), f"replay {i}"


def test_after_controls(S):
    """As a server runs them: controls, then the choice; a row whose mask allows nothing answers -1."""
    from ossm_amd.logits import control_logits, pack_allowed

    rows, V = 4, 1000
    x = torch.randn(rows, V).cuda()
    hist = torch.randint(0, V, (rows, 50), dtype=torch.int32).cuda()
    allowed = torch.rand(rows, V).cuda() < 0.2
    allowed[2] = False
    announce("sample_logits after control_logits")
    y = control_logits(x, hist, repetition=1.3, frequency=0.2, allowed=pack_allowed(allowed))
    for t in (1.0, 0.0):
        got = check(S, y, np.random.default_rng(4).random(rows), t, 50, 0.9)
        assert got[2] == -1 and all(allowed[i, got[i]] for i in (0, 1, 3))


def test_refusals(S):
    x, u = torch.zeros(2, 40).cuda(), torch.zeros(2).cuda()
    for match, kw in (("logits must be", {"logits": x.half()}), ("logits must be", {"logits": x.cpu()}),
                      ("logits must be", {"logits": x[0]}), ("uniform must be", {"uniform": u.double()}),
                      ("uniform must be", {"uniform": u[:1]}), ("uniform must be", {"uniform": u.cpu()}),
                      ("1 to 2\\^20", {"logits": x[:, :0]}), ("temperature must be", {"temperature": u.double()}),
                      ("temperature must be", {"temperature": "hot"}), ("top_p must be", {"top_p": u[:1]}),
                      ("min_p must be", {"min_p": x}), ("top_k must be", {"top_k": u}),
                      ("top_k must be", {"top_k": torch.zeros(3, dtype=torch.int32).cuda()}),
                      ("out must be", {"out": torch.zeros(2, dtype=torch.int32).cuda()}),
                      ("out must be", {"out": torch.zeros(3, dtype=torch.int64).cuda()})):
        with pytest.raises(RuntimeError, match=match):
            S.sample_logits(**{"logits": x, "uniform": u, **kw})
    assert S.sample_logits(x[:0], u[:0]).shape == (0,)


def below_the_bins():
    """Rows of which a large top-k reaches entries that weigh nothing: masked with finite values, or
    far below at a low temperature.  (name, row, temperature, k)"""
    rng = np.random.default_rng(93)

    def masked(allowed, others, value):
        row = np.full(allowed + others, value)
        row[rng.permutation(allowed + others)[:allowed]] = rng.normal(size=allowed)
        return row

    return [("masked -1e9", masked(900, 3600, -1e9), 1.0, 1000), ("masked -1e4", masked(5000, 3000, -1e4), 1.0, 6000),
            ("masked -1e9, most allowed", masked(5000, 1000, -1e9), 1.0, 5500), ("masked lowest", masked(5000, 1000, -3.38e38), 1.0, 5001),
            ("masked, k the last", masked(4200, 400, -1e9), 2.0, 4599), ("low temperature", rng.normal(size=5000) * 3, 0.3, 4500),
            ("lower temperature", rng.normal(size=8000), 0.13, 7990)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", range(7))
def test_top_k_past_what_weighs_anything(S, case, dtype):
    name, row, t, k = below_the_bins()[case]
    announce(f"sample_logits {name} {dtype}")
    n = 20
    x = torch.tensor(np.stack([row] * n)).to(dtype).cuda()
    u = (np.arange(n) + 0.5) / n
    part = np.array([0.05, 0.5, 0.9, 0.999] * 5)
    for kw in ({}, {"top_p": part}, {"min_p": 0.2}, {"top_p": part, "min_p": 0.01}):
        out = torch.full((n,), -77, dtype=torch.int64, device="cuda")
        check(S, x, u, t, k, out=out, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_rows_whose_every_eighth_entry_is_alike(S, dtype):
    """Every eighth entry within 1e-27 of the largest and the others 1e13 below, at a temperature at which they
    weigh as much: top-k counts them all."""
    V, n = 8000, 16
    row = np.full(V, -1e13)
    row[::8] = 0.0
    row[0] = 1e-27
    x = torch.tensor(np.stack([row] * n)).to(dtype).cuda()
    u = np.append((np.arange(n - 1) + 0.5) / n, 1 - 2.0 ** -24)
    announce(f"sample_logits every eighth alike {dtype}")
    for k in (1000, 1001, 5000, 7999):
        check(S, x, u, 1e13, k)
        check(S, x, u, 1e14, k, 0.9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_parts_next_to_one(S, dtype):
    """A top-p whose border lies in the tail of a large vocabulary, past what a list holds."""
    announce(f"sample_logits p next to one {dtype}")
    rng = np.random.default_rng(94)
    part = np.array([0.9995, 0.99999, 1 - 2.0 ** -24, 0.9994, 0.9996, 0.999])
    for V in (50001, 131072):
        x = torch.tensor(rng.normal(size=(6, V)) * 1.5).to(dtype).cuda()
        for u in (rng.random(6), np.full(6, 1 - 2.0 ** -24)):
            check(S, x, u, 1.0, 0, part)
            check(S, x, u, 1.3, V - 100, part)
            check(S, x, u, 1.0, 0, part, 1e-5)


def test_random_numbers_at_the_borders_of_unequal_weights(S):
    """u next to each running sum of unequal weights, below and above: the token before and the one
    after.  The kernel's sums are off by less than 4 units of 2^-46 of the largest weight; no u is that
    near a sum, which is checked in extended precision first."""
    for values in ([1.0, 2.0, 4.0, 1.0], [3.0, 5.0, 7.0, 0.01, 11.0, 1e-4], [0.3, 0.2, 0.1]):
        row = np.log(np.array(values)).astype(np.float32).astype(np.longdouble)
        w = np.exp(row - row.max())
        cum = np.cumsum(w) / w.sum()
        below = np.array([np.float32(c) if np.float32(c) < c else np.nextafter(np.float32(c), np.float32(0)) for c in cum[:-1]])
        u = np.stack([below, np.nextafter(below, np.float32(1))], 1).reshape(-1)
        assert np.abs(u[:, None].astype(np.longdouble) - cum[None]).min() > 2.0 ** -40
        want = [i // 2 + i % 2 for i in range(2 * len(below))]
        x = torch.tensor(np.stack([row] * len(u)).astype(np.float32)).cuda()
        announce(f"sample_logits at the borders of {values}")
        assert check(S, x, u).tolist() == want
        assert check(S, x, u, 1.0, len(values)).tolist() == want
