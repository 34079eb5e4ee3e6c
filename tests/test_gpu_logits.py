"""GPU tests of control_logits against a float64 row-by-row computation.

Tolerances, derived before the first run: a logit takes one product or division, at
most two subtractions of exact multiples and one addition in float32, so 4 roundings
of 2^-24 of the largest value on the way (|l| * rep + |freq c + pres| + |bias|);
a bfloat16 output adds half an ulp, 2^-9 (2^-8 leaves room for a neighbour's tie)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    need_gpu()
    from ossm_amd import logits

    return logits


def reference(logits, hist, n, first, rep, pres, freq, ids, vals, allowed):
    """(result, size on the way) in float64."""
    out = logits.double().cpu().numpy().copy()
    size = np.abs(out)
    S, V = out.shape
    for i in range(S):
        row = out[i]
        h = hist[i, :n[i]] if hist is not None else np.zeros(0, int)
        said = hist[i, first[i]:n[i]] if hist is not None else np.zeros(0, int)
        for v in np.unique(h):
            if 0 <= v < V:
                row[v] = row[v] / rep[i] if row[v] > 0 else row[v] * rep[i]
        size[i] = np.maximum(size[i], np.abs(row))
        said = said[(said >= 0) & (said < V)]
        c = np.bincount(said, minlength=V)
        row -= np.where(c > 0, freq[i] * c + pres[i], 0)
        size[i] += np.abs(freq[i] * c + pres[i])
        if ids is not None:
            last = {int(t): float(x) for t, x in zip(ids[i], vals[i]) if 0 <= t < V}
            for t, x in last.items():
                row[t] += x
                size[i, t] += abs(x)
        if allowed is not None:
            row[~allowed[i]] = -np.inf
    return out, size


def check(got, want, size, dtype):
    g = got.double().cpu().numpy()
    same = (g == want) | (np.isnan(g) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        tol = 4 * 2.0 ** -24 * size + (2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0)
        bad = ~(same | (np.abs(g - want) <= tol))
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, first at {np.argwhere(bad)[0]}"


def inputs(S, V, H, Kb, dtype, seed, mask=True):
    rng = np.random.default_rng(seed)
    x = torch.tensor(rng.normal(size=(S, V)) * 3, dtype=dtype).cuda()
    hist = (rng.random((S, H)) ** 4 * V).astype(np.int32)
    hist[rng.random((S, H)) < 0.05] = -1           # padding
    hist[rng.random((S, H)) < 0.05] = V + 7        # outside
    n = rng.integers(0, H + 1, S)
    first = rng.integers(0, H + 1, S)
    ids = rng.integers(-1, V, (S, Kb)).astype(np.int32)
    if Kb >= 2:
        ids[:, -1] = ids[:, 0]                     # given twice: the last counts
    vals = (rng.normal(size=(S, Kb)) * 5).astype(np.float32)
    rep, pres, freq = (rng.uniform(a, b, S).astype(np.float32) for a, b in ((0.8, 1.6), (-1, 1), (-0.3, 0.5)))
    allowed = rng.random((S, V)) < 0.3 if mask else None
    if mask:
        allowed[0] = False                         # a row that may answer nothing
    return x, hist, n, first, rep, pres, freq, ids, vals, allowed


def call(L, x, hist, n, first, rep, pres, freq, ids, vals, allowed, **kw):
    t = lambda a: None if a is None else torch.tensor(a).cuda()  # noqa: E731
    return L.control_logits(x, t(hist), t(n), t(first), repetition=t(rep), presence=t(pres), frequency=t(freq),
                            bias_ids=t(ids), bias_values=t(vals),
                            allowed=None if allowed is None else L.pack_allowed(t(allowed)), **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (3, 31, 0, 0), (2, 33, 5, 2), (5, 1000, 700, 3), (4, 8191, 50, 7),
                                  (3, 8192, 1, 0), (7, 8193, 300, 40), (2, 50001, 2000, 300), (33, 4099, 64, 16),
                                  (2, 300, 70000, 5), (1, 9000, 20, 70000)],
                         ids=lambda s: "x".join(map(str, s)))
def test_matches_float64(L, size, dtype):
    announce(f"control_logits {size} {dtype}")
    a = inputs(*size, dtype, seed=size[1])
    want, sz = reference(*a)
    check(call(L, *a), want, sz, dtype)
    inplace = a[0].clone()
    assert call(L, inplace, *a[1:], out=inplace) is inplace
    check(inplace, want, sz, dtype)


def test_parts_alone_and_numbers_for_all_rows(L):
    S, V, H = 4, 777, 60
    x, hist, n, first, rep, pres, freq, ids, vals, allowed = inputs(S, V, H, 5, torch.float32, 1)
    ones, zeros, full = np.ones(S), np.zeros(S), np.full(S, H)
    none = (None, None, None)
    announce("control_logits parts alone")
    assert torch.equal(L.control_logits(x), x)
    h = torch.tensor(hist).cuda()
    want = reference(x, hist, full, zeros.astype(int), np.full(S, np.float32(1.2)), ones * 0.5, ones * 0.25, *none)
    check(L.control_logits(x, h, repetition=np.float32(1.2).item(), presence=0.5, frequency=0.25), *want, torch.float32)
    want = reference(x, None, full, full, ones, zeros, zeros, ids, vals, None)
    check(L.control_logits(x, bias_ids=torch.tensor(ids).cuda(), bias_values=torch.tensor(vals).cuda()), *want,
          torch.float32)
    one = np.repeat(allowed[1:2], S, 0)
    want = reference(x, None, full, full, ones, zeros, zeros, None, None, one)
    check(L.control_logits(x, allowed=L.pack_allowed(torch.tensor(allowed[1]).cuda())), *want, torch.float32)
    # one row of biases for all, with each row's values
    same = np.repeat(ids[:1], S, 0)
    want = reference(x, None, full, full, ones, zeros, zeros, same, vals, None)
    check(L.control_logits(x, bias_ids=torch.tensor(ids[0]).cuda(), bias_values=torch.tensor(vals).cuda()), *want,
          torch.float32)


def test_special_values(L):
    """Masked places are -inf whatever they held; others keep NaN and infinities; the
    type's lowest value is a value like others."""
    V = 100
    x = torch.zeros(3, V).cuda()
    low = torch.finfo(torch.float32).min
    x[0, :5] = torch.tensor([float("nan"), float("inf"), -float("inf"), low, -0.0]).cuda()
    x[1] = low
    x[2] = float("nan")
    allowed = torch.ones(3, V, dtype=torch.bool).cuda()
    allowed[0, 0] = allowed[0, 1] = False
    allowed[2] = False
    hist = torch.tensor([[2, 3, 4], [0, 0, 1], [1, 2, 3]], dtype=torch.int32).cuda()
    announce("control_logits special values")
    y = L.control_logits(x, hist, repetition=2.0, allowed=L.pack_allowed(allowed))
    assert y[0, 0] == -float("inf") and y[0, 1] == -float("inf") and y[0, 2] == -float("inf")
    assert y[0, 3] == -float("inf") and y[0, 4] == 0  # twice the lowest value overflows
    assert y[1, 0] == -float("inf") and y[1, 5] == low
    assert torch.all(y[2] == -float("inf"))
    y = L.control_logits(x, hist, presence=1.0)
    assert torch.isnan(y[0, 0]) and y[0, 1] == float("inf") and torch.isnan(y[2]).all() and y[1, 0] == low


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides_offsets_and_other_streams(L, dtype):
    """Rows at every 16-byte offset, a wide row stride, an output at another offset, and a
    side stream: all bitwise what dense tensors give."""
    S, V = 5, 9001
    a = inputs(S, V, 100, 9, dtype, 3)
    want = call(L, *a)
    for off in range(9):
        wide = torch.zeros(S, V + 40, dtype=dtype, device="cuda")
        view = wide[:, off:off + V]
        view.copy_(a[0])
        out = torch.full((S, V + 23), 7.0, dtype=dtype, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        announce(f"control_logits offset {off} {dtype}")
        with torch.cuda.stream(side):
            got = call(L, view, *a[1:], out=out[:, off % 3:off % 3 + V])
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        rest = torch.ones(V + 23, dtype=torch.bool)
        rest[off % 3:off % 3 + V] = False
        assert torch.all(out[:, rest.cuda()] == 7)


def test_logits_past_32_bits(L):
    """Rows that start past 2^31 elements."""
    S, V = 11000, 200003
    assert (S - 1) * V > 2 ** 31
    x = torch.empty(S, V, dtype=torch.bfloat16, device="cuda")
    a = inputs(2, V, 50, 4, torch.bfloat16, 4)
    x[-2:] = a[0]
    want, sz = reference(*a)
    grow = lambda t: None if t is None else np.concatenate([np.zeros((S - 2, *t.shape[1:]), t.dtype), t])  # noqa: E731
    big = [grow(t) for t in a[1:9]]
    announce("control_logits past 2^31 elements")
    t = [torch.tensor(b).cuda() for b in big]
    mask = torch.zeros(S, (V + 31) // 32, dtype=torch.int32, device="cuda")
    mask[-2:] = L.pack_allowed(torch.tensor(a[9]).cuda())
    L.control_logits(x, t[0], t[1], t[2], repetition=t[3], presence=t[4], frequency=t[5], bias_ids=t[6],
                     bias_values=t[7], allowed=mask, out=x)
    check(x[-2:], want, sz, torch.bfloat16)


def test_graph_capture(L):
    x, *rest = inputs(3, 5000, 100, 4, torch.float32, 5)
    t = lambda a: torch.tensor(a).cuda()  # noqa: E731
    hist, n, first, rep, pres, freq, ids, vals = (t(a) for a in rest[:8])
    n, first, mask = n.to(torch.int32), first.to(torch.int32), L.pack_allowed(t(rest[8]))
    run = lambda v: L.control_logits(v, hist, n, first, repetition=rep, presence=pres, frequency=freq,  # noqa: E731
                                     bias_ids=ids, bias_values=vals, allowed=mask)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    announce("control_logits under graph capture")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = run(x)
    for i in range(4):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, run(x)), f"replay {i}"


def test_refusals(L):
    x = torch.zeros(2, 40).cuda()
    h = torch.zeros(2, 3, dtype=torch.int32).cuda()
    for match, kw in (("float32 or bfloat16", {"logits": x.half()}), ("history must be", {"history": h.long()}),
                      ("history must be", {"history": h[:, 0]}), ("lengths must be", {"history": h, "lengths": h}),
                      ("without a history", {"lengths": h[:, 0]}), ("repetition must be", {"repetition": x[0]}),
                      ("both bias_ids", {"bias_ids": h}), ("allowed must be", {"allowed": h}),
                      ("bias_values must be", {"bias_ids": h, "bias_values": x}),
                      ("out must have", {"out": x.bfloat16()}), ("out must have", {"out": x.t()}),
                      ("allowed must be", {"allowed": torch.zeros(2, 2, dtype=torch.int32)}),
                      ("inference", {"logits": x.clone().requires_grad_(True)}),
                      ("logits must be", {"logits": x[0]}), ("logits must be", {"logits": x.cpu()})):
        with pytest.raises(RuntimeError, match=match):
            L.control_logits(**{"logits": x, **kw})


@torch.random.fork_rng()  # later tests draw what they drew
def test_forward_mode_is_refused(L):
    """A tangent raises, under no_grad too, whichever argument carries it."""
    from torch.autograd import forward_ad

    floats = {"logits": torch.randn(2, 40).cuda(), "bias_values": torch.randn(2, 3).cuda(),
              **{k: torch.ones(2).cuda() for k in ("repetition", "presence", "frequency")}}
    ids = torch.arange(3, dtype=torch.int32).cuda()[None]
    announce("control_logits with tangents")
    L.control_logits(**floats, bias_ids=ids)
    for k, t in floats.items():
        with torch.no_grad(), forward_ad.dual_level(), pytest.raises(RuntimeError, match="tangents"):
            L.control_logits(**{**floats, k: forward_ad.make_dual(t, torch.ones_like(t))}, bias_ids=ids)


@torch.random.fork_rng()  # later tests draw what they drew
def test_gradients_are_refused(L):
    """Of the logits and of every penalty and bias, where one is wanted."""
    floats = {"logits": torch.randn(2, 40).cuda(), "bias_values": torch.randn(2, 3).cuda(),
              **{k: torch.ones(2).cuda() for k in ("repetition", "presence", "frequency")}}
    ids = torch.arange(3, dtype=torch.int32).cuda()[None]
    announce("control_logits with gradients")
    for k, t in floats.items():
        grad = {**floats, k: t.clone().requires_grad_(True)}
        with pytest.raises(RuntimeError, match="inference"):
            L.control_logits(**grad, bias_ids=ids)
        with torch.no_grad():
            L.control_logits(**grad, bias_ids=ids)


def test_a_vocabulary_of_one_at_any_stride(L):
    """A single column has no column stride to check, in place too."""
    wide = torch.arange(1.0, 41.0).cuda().view(5, 8)
    x, out = wide[:, 2:3].T.T, wide[:, ::3][:, 2:3]
    one = torch.as_strided(wide, (5, 1), (8, 3), 4)
    announce("control_logits of one column, strided")
    want = one.clone() * 0.5
    hist = torch.zeros(1, 1, dtype=torch.int32).cuda()
    assert L.control_logits(one, hist, repetition=2.0, out=one) is one
    assert torch.equal(one, want)
    assert torch.equal(L.control_logits(x, hist, repetition=2.0, out=out), x * 0.5)
