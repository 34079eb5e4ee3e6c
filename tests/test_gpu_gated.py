"""GPU tests of the gated projection (ossm_amd.gated), forward and backward, against
float64 formulas, and of its gradients against differences.

Tolerances, derived before the first run.  float32: products of K terms keep 24
bits of each factor and are summed in float32, so an output is off by at most about
sqrt(K) 2^-24 of the sum of |terms|'s size (a random walk; 4 of them bound it), and
the activation's own error of a few 2^-22: 1e-5 of the tensor's largest value covers
K up to 10^4.  bfloat16: one rounding of the output, 2^-8 of it (half an ulp and a
neighbour's tie); in the backward the stored a and b and the rounded da and db each add
a relative 2^-9 to every term, random, so 4 * 2^-9 of the root of the sum of the terms'
squares, below 2^-6 of the gradient's largest value."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh", "sigmoid", "relu"]


@pytest.fixture(scope="module")
def G():
    need_gpu()
    from ossm_amd import gated

    return gated


def act64(name, a):
    """The activation and its derivative, in float64."""
    s = 1 / (1 + np.exp(-a))
    if name == "silu":
        return a * s, s * (1 + a * (1 - s))
    if name == "sigmoid":
        return s, s * (1 - s)
    if name == "relu":
        return np.maximum(a, 0), (a > 0) * 1.0
    if name == "gelu":
        cdf = 0.5 * (1 + np.vectorize(math.erf)(a / math.sqrt(2)))
        return a * cdf, cdf + a * np.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = np.tanh(c * (a + 0.044715 * a ** 3))
    return 0.5 * a * (1 + t), 0.5 * (1 + t) + 0.5 * a * (1 - t * t) * c * (1 + 3 * 0.044715 * a * a)


def reference(x, wg, wu, bg, bu, act, go=None):
    x, wg, wu, bg, bu, go = (None if t is None else t.detach().double().cpu().numpy() for t in (x, wg, wu, bg, bu, go))
    a, b = x @ wg.T, x @ wu.T
    if bg is not None:
        a = a + bg
    if bu is not None:
        b = b + bu
    f, d = act64(act, a)
    if go is None:
        return f * b
    da, db = go * b * d, go * f
    return [f * b, da @ wg + db @ wu, da.T @ x, db.T @ x, da.sum(0), db.sum(0)]


def inputs(T, D, n, dtype, bias, seed=0, scale=2.0):
    rng = np.random.default_rng(seed)
    f = lambda *s, k=1.0: torch.tensor(rng.normal(size=s) * k, dtype=torch.float32).to(dtype).cuda()  # noqa: E731
    k = scale / math.sqrt(max(D, 1))
    return [f(T, D), f(n, D, k=k), f(n, D, k=k), f(n) if bias else None, f(n) if bias else None], f(T, n)


def check(got, want, dtype, what, gradient=False):
    g = got.detach().double().cpu().numpy()
    assert g.shape == want.shape, what
    top = np.abs(want).max(initial=0)
    tol = 1e-5 * top + (0 if dtype == torch.float32 else 2.0 ** -8 * np.abs(want) + (2.0 ** -6 * top if gradient else 0))
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())}/{bad.size} off, worst {np.abs(g - want).max():.3e} of {top:.3e}"


# T, D, F: one row to several tiles, sizes that are no multiple of 8, 32 or the tiles
SHAPES = [(1, 1, 1), (1, 64, 32), (2, 7, 5), (3, 8, 9), (5, 2048, 130), (16, 128, 512), (17, 100, 33), (33, 65, 129),
          (64, 72, 200), (65, 640, 257), (130, 258, 131), (257, 96, 520), (1000, 128, 172), (300, 1024, 1030)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward_match_float64(G, shape, dtype):
    for i, act in enumerate(ACTS):
        bias = i % 2 == 0
        args, go = inputs(*shape, dtype, bias, seed=i)
        want = reference(*args, act, go)
        announce(f"gated_linear {shape} {dtype} {act} bias={bias}")
        with torch.no_grad():
            check(G.gated_linear(*args, activation=act), want[0], dtype, f"{act} y")
        leaves = [t.requires_grad_(True) for t in args if t is not None]
        y = G.gated_linear(*args, activation=act)
        check(y, want[0], dtype, f"{act} y, training")
        for g, w, n in zip(torch.autograd.grad(y, leaves, go), want[1:], ("x", "gate", "up", "gate bias", "up bias")):
            check(g, w, dtype, f"{act} grad {n}", True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_large_tiles(G, dtype):
    """Enough tiles for the largest workgroups, both ways, and ragged ends."""
    for shape in ((4100, 136, 2056), (2100, 2050, 264)):
        args, go = inputs(*shape, dtype, False, seed=3)
        announce(f"gated_linear large tiles {shape} {dtype}")
        want = reference(*args, "silu", go)
        leaves = [t.requires_grad_(True) for t in args[:3]]
        y = G.gated_linear(*args)
        check(y, want[0], dtype, "y")
        for g, w, n in zip(torch.autograd.grad(y, leaves, go), want[1:], ("x", "gate", "up")):
            check(g, w, dtype, f"grad {n}", True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(513, 40, 70), (520, 130, 33), (700, 264, 40), (1025, 7, 5)],
                         ids=lambda s: "x".join(map(str, s)))
def test_forward_past_few_rows(G, shape, dtype):
    """Products over the whole batch, however small."""
    for i, act in enumerate(ACTS):
        args, _ = inputs(*shape, dtype, i % 2 == 0, seed=20 + i)
        announce(f"gated_linear products {shape} {dtype} {act}")
        with torch.no_grad():
            check(G.gated_linear(*args, activation=act), reference(*args, act), dtype, act)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_values_that_are_not_finite_past_few_rows(G, dtype):
    args, _ = inputs(600, 40, 70, dtype, False, seed=21)
    x, wg, wu = args[:3]
    base = G.gated_linear(x, wg, wu, activation="relu")
    for value in (float("inf"), -float("inf"), float("nan")):
        xi, wi = x.clone(), wu.clone()
        xi[1, 3] = value
        wi[69, 5] = value
        announce(f"gated_linear {value} rows=600 {dtype}")
        y = G.gated_linear(xi, wg, wi, activation="relu")
        keep = [i for i in range(600) if i != 1]
        assert torch.equal(y[keep][:, :69], base[keep][:, :69])
        want = reference(xi, wg, wi, None, None, "relu")
        g = y.double().cpu().numpy()
        assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(np.isposinf(g), np.isposinf(want))
        assert np.array_equal(np.isneginf(g), np.isneginf(want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_few_rows_of_any_alignment(G, dtype):
    """Rows and sizes at every offset, D from below a block to several, several groups of rows."""
    for T, D, n in ((1, 31, 17), (15, 33, 16), (16, 128, 40), (31, 300, 15), (33, 2050, 48), (63, 513, 31), (127, 1025, 50),
                    (200, 1000, 70)):
        args, _ = inputs(T, D, n, dtype, True, seed=T)
        want = reference(*args, "silu")
        for off in (0, 1, 3, 8):
            wide = [torch.full((t.size(0), D + 11), float("nan"), dtype=dtype, device="cuda") for t in args[:3]]
            for w, t in zip(wide, args):
                w[:, off:off + D] = t
            announce(f"gated_linear few rows {T} {D} {n} offset {off} {dtype}")
            with torch.no_grad():
                y = G.gated_linear(*(w[:, off:off + D] for w in wide), *args[3:])
            check(y, want, dtype, f"offset {off}")


@pytest.mark.parametrize("shape", [(1, 100, 64), (1, 256, 2000), (2, 64, 4096), (40, 33, 70), (5, 130, 600)],
                         ids=lambda s: "x".join(map(str, s)))
def test_few_gradients_lose_nothing_before_their_rounding(G, shape):
    """bfloat16, few da and db: what is off is the rounding of the result alone.  It moves a
    value by at most 2^-8 of it, uniformly, so by at most 2^-8 / sqrt(3) in the root mean
    square; a twentieth more is room for chance and the float32 sums."""
    for seed, act in enumerate(ACTS * 2):
        args, go = inputs(*shape, torch.bfloat16, False, seed=40 + seed)
        announce(f"gated_linear few gradients {shape} {act}")
        want = reference(*args, act, go)[1:4]
        leaves = [t.requires_grad_(True) for t in args[:3]]
        for g, w, n in zip(torch.autograd.grad(G.gated_linear(*leaves, activation=act), leaves, go), want, ("x", "gate", "up")):
            off = np.sqrt(((g.double().cpu().numpy() - w) ** 2).sum() / (w ** 2).sum())
            assert off <= 1.05 * 2.0 ** -8 / math.sqrt(3), f"{act} grad {n}: {off:.5f}"


def test_few_gradients_of_infinite_weights(G):
    """An infinite weight reaches x's gradient in its column alone, as an infinity."""
    args, go = inputs(3, 40, 70, torch.bfloat16, False, seed=60)
    announce("gated_linear gradient through an infinite weight")
    go[:] = 1
    x, wg, wu = (t.requires_grad_(True) for t in args[:3])
    y = G.gated_linear(x, wg, wu, activation="sigmoid")
    wu.data[7, 5] = float("inf")  # db = sigmoid(a) > 0
    g = torch.autograd.grad(y, [x], go)[0]
    assert torch.isposinf(g[:, 5]).all() and torch.isfinite(g[:, :5]).all() and torch.isfinite(g[:, 6:]).all()


def test_gradients_against_differences(G):
    """Central differences of a random projection of y, along random directions."""
    (args, go) = inputs(40, 24, 50, torch.float32, True, seed=4)
    for act in ACTS[:4]:  # relu has a corner
        leaves = [t.clone().requires_grad_(True) for t in args]
        announce(f"gated_linear differences {act}")
        grads = torch.autograd.grad(G.gated_linear(*leaves, activation=act), leaves, go)
        for i, (t, g) in enumerate(zip(args, grads)):
            v = torch.randn_like(t)
            h = 2.0 ** -7  # truncation h^2 f''' / 6, rounding 2^-24 |f| / h: both near 1e-5 of the sum's size
            hi, lo = ([p + s * h * v if j == i else p for j, p in enumerate(args)] for s in (1, -1))
            with torch.no_grad():
                d = G.gated_linear(*hi, activation=act).double() - G.gated_linear(*lo, activation=act).double()
            terms = d * go.double() / (2 * h)
            assert abs(terms.sum() - (g.double() * v.double()).sum()) <= 1e-3 * terms.abs().sum()


def test_second_derivatives_and_partial_needs(G):
    args, go = inputs(20, 16, 24, torch.float32, True, seed=5)
    leaves = [t.requires_grad_(True) for t in args]
    announce("gated_linear twice differentiated")
    g = torch.autograd.grad(G.gated_linear(*leaves), leaves, go, create_graph=True)
    got = torch.autograd.grad(sum((t * t).sum() for t in g), leaves)
    ref = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    y = torch.nn.functional.silu(ref[0] @ ref[1].t() + ref[3]) * (ref[0] @ ref[2].t() + ref[4])
    g = torch.autograd.grad(y, ref, go.double().cpu(), create_graph=True)
    for a, b in zip(got, torch.autograd.grad(sum((t * t).sum() for t in g), ref)):
        assert torch.allclose(a.double().cpu(), b, rtol=1e-4, atol=1e-4 * float(b.abs().max()))
    for keep in range(5):
        part = [t.detach().requires_grad_(i == keep) for i, t in enumerate(leaves)]
        (got,) = torch.autograd.grad(G.gated_linear(*part), [part[keep]], go)
        check(got, reference(*part, "silu", go)[1 + keep], torch.float32, f"only input {keep}", True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [3, 40, 300])
def test_values_that_are_not_finite(G, rows, dtype):
    """An infinity or NaN reaches its own row (x) or column (weight), with the right sign,
    and nothing else; the largest float32 values are values like others."""
    args, _ = inputs(rows, 40, 70, dtype, False, seed=6)
    x, wg, wu = args[:3]
    base = G.gated_linear(x, wg, wu, activation="relu")
    for value in (float("inf"), -float("inf"), float("nan")):
        xi, wi = x.clone(), wu.clone()
        xi[1, 3] = value
        wi[69, 5] = value
        announce(f"gated_linear {value} rows={rows} {dtype}")
        y = G.gated_linear(xi, wg, wi, activation="relu")
        keep_r, keep_c = [i for i in range(rows) if i != 1], list(range(69))
        assert torch.equal(y[keep_r][:, keep_c], base[keep_r][:, keep_c])
        want = reference(xi, wg, wi, None, None, "relu")
        g = y.double().cpu().numpy()
        assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(np.isposinf(g), np.isposinf(want))
        assert np.array_equal(np.isneginf(g), np.isneginf(want))
    big = torch.zeros_like(x)
    big[0, 0] = torch.finfo(dtype).max
    one = torch.zeros_like(wg)
    one[:, 0] = 1
    half = torch.zeros_like(wu)
    half[:, 0] = 2.0 ** -64
    y = G.gated_linear(big, one, half, None, torch.full((70,), 0.0, dtype=dtype, device="cuda"), activation="sigmoid")
    check(y, reference(big, one, half, None, None, "sigmoid"), dtype, "largest value")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides_leading_dimensions_and_streams(G, dtype):
    args, go = inputs(60, 64, 96, dtype, True, seed=7)
    x, wg, wu, bg, bu = args
    with torch.no_grad():
        want = G.gated_linear(*args)
        wide = torch.full((60, 200), float("nan"), dtype=dtype, device="cuda")
        for off in (0, 1, 8, 72):
            wide[:, off:off + 64] = x
            announce(f"gated_linear strided offset {off} {dtype}")
            assert torch.equal(G.gated_linear(wide[:, off:off + 64], wg, wu, bg, bu), want)
        wt = wg.t().contiguous().t()
        both = torch.cat([wg, wu], 1)
        assert torch.equal(G.gated_linear(x, wt, wu, bg, bu), want)
        assert torch.equal(G.gated_linear(x, both[:, :64], both[:, 64:], bg, bu), want)
        assert torch.equal(G.gated_linear(x.view(3, 4, 5, 64), *args[1:]), want.view(3, 4, 5, 96))
        assert torch.equal(G.gated_linear(x[:1].expand(60, 64), *args[1:]), want[:1].expand(60, 96))
        assert torch.equal(G.gated_linear(x[5], *args[1:]), G.gated_linear(x[5:6], *args[1:])[0])
    leaves = [t.requires_grad_(True) for t in args]
    first = torch.autograd.grad(G.gated_linear(*leaves), leaves, go)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(G.gated_linear(*leaves), leaves, go.t().contiguous().t())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))  # and bitwise repeatable
    one = torch.ones((), dtype=dtype, device="cuda")
    wide = torch.autograd.grad(G.gated_linear(*leaves).sum(), leaves)
    dense = torch.autograd.grad(G.gated_linear(*leaves), leaves, one.expand(60, 96).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(wide, dense))  # a broadcast gradient


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(626, 1954, 86), (1679, 1549, 94), (530, 2048, 264), (2161, 600, 1)],
                         ids=lambda s: "x".join(map(str, s)))
def test_few_tiles_share_k(G, shape, dtype):
    """Long products of few tiles: with and without biases and saved projections."""
    for bias, act in ((True, "sigmoid"), (False, "gelu")):
        args, go = inputs(*shape, dtype, bias, seed=30)
        want = reference(*args, act, go)
        announce(f"gated_linear shared k {shape} {dtype} {act} bias={bias}")
        with torch.no_grad():
            y = G.gated_linear(*args, activation=act)
            check(y, want[0], dtype, act)
            assert torch.equal(y, G.gated_linear(*args, activation=act))
        leaves = [t.requires_grad_(True) for t in args if t is not None]
        y = G.gated_linear(*args, activation=act)
        check(y, want[0], dtype, "y, training")
        for g, w, n in zip(torch.autograd.grad(y, leaves, go), want[1:], ("x", "gate", "up", "gate bias", "up bias")):
            check(g, w, dtype, f"{act} grad {n}", True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_values_that_are_not_finite_among_few_tiles(G, dtype):
    """An infinite and a NaN input reach their own rows and no other's bits."""
    args, _ = inputs(700, 1100, 70, dtype, False, seed=31)
    x, wg, wu = args[:3]
    announce(f"gated_linear shared k, not finite {dtype}")
    base = G.gated_linear(x, wg, wu, activation="sigmoid")
    bad = x.clone()
    bad[5, 1090] = float("nan")
    bad[650, 3] = float("inf")
    got = G.gated_linear(bad, wg, wu, activation="sigmoid")
    keep = [r for r in range(700) if r not in (5, 650)]
    assert torch.equal(got[keep], base[keep])
    assert got[5].isnan().all()
    # sigmoid(+-inf) of +-inf: 0 inf is NaN, 1 inf is inf with the up weight's sign
    g, u = wg[:, 3].float(), wu[:, 3].float()
    want = torch.where(g > 0, u.sign() * float("inf"), float("nan"))
    assert torch.equal(got[650].float().nan_to_num(7.0, 8.0, -8.0), want.nan_to_num(7.0, 8.0, -8.0))


def test_rows_past_32_bits(G):
    """More outputs than 32 bits count; gradients only in the first and last rows, whose
    float64 formulas give all there is of the weights'."""
    T, D, n, ends = (1 << 20) + 77, 32, 2056, 40
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(T, D, device="cuda", generator=g).bfloat16()
    wg, wu = (torch.randn(n, D, device="cuda", generator=g).mul(2 / math.sqrt(D)).bfloat16() for _ in range(2))
    rows = torch.cat([torch.arange(ends), torch.arange(T - ends, T)]).cuda()
    go = torch.zeros(T, n, dtype=torch.bfloat16, device="cuda")
    go[rows] = torch.randn(2 * ends, n, device="cuda", generator=g).bfloat16()
    want = reference(x[rows], wg, wu, None, None, "silu", go[rows])
    announce(f"gated_linear past 32 bits {(T, D, n)}")
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    y = G.gated_linear(*leaves)
    check(y[rows], want[0], torch.bfloat16, "y")
    gx, *gw = torch.autograd.grad(y, leaves, go)
    check(gx[rows], want[1], torch.bfloat16, "grad x", True)
    assert not gx[ends:T - ends].any()
    for got, w, name in zip(gw, want[2:], ("gate", "up")):
        check(got, w, torch.bfloat16, f"grad {name}", True)


def test_empty(G):
    z = lambda *s: torch.zeros(*s, device="cuda", requires_grad=True)  # noqa: E731
    announce("gated_linear empty")
    for T, D, n in ((0, 8, 5), (4, 8, 0), (0, 0, 0)):
        x, wg, wu = z(T, D), z(n, D), z(n, D)
        y = G.gated_linear(x, wg, wu)
        assert y.shape == (T, n)
        for g, t in zip(torch.autograd.grad(y, [x, wg, wu], torch.ones_like(y)), (x, wg, wu)):
            assert g.shape == t.shape and torch.all(g == 0)
    b = torch.randn(6, device="cuda", requires_grad=True)
    x, wg, wu = z(4, 0), z(6, 0), z(6, 0)
    y = G.gated_linear(x, wg, wu, b, b, "sigmoid")  # biases only
    assert torch.allclose(y, (torch.sigmoid(b) * b).expand(4, 6), rtol=1e-6)
    (gb,) = torch.autograd.grad(y, [b], torch.ones_like(y))
    s = torch.sigmoid(b.detach())
    assert torch.allclose(gb, 4 * (s + b.detach() * s * (1 - s)), rtol=1e-5, atol=1e-6)


def test_graph_capture(G):
    args, go = inputs(100, 200, 60, torch.bfloat16, True, seed=8)
    leaves = [t.requires_grad_(True) for t in args]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    announce("gated_linear under graph capture")
    with torch.cuda.stream(side):
        torch.autograd.grad(G.gated_linear(*leaves), leaves, go)  # the workspace grows before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = G.gated_linear(*leaves)
        grads = torch.autograd.grad(y, leaves, go)
    for i in range(4):
        with torch.no_grad():
            args[0].normal_()
        graph.replay()
        torch.cuda.synchronize()
        y2 = G.gated_linear(*leaves)
        assert torch.equal(y, y2)
        assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(y2, leaves, go))), f"replay {i}"


def test_module_and_autocast(G):
    torch.manual_seed(0)
    m = G.GatedFeedForward(48, 100, activation="gelu").cuda()
    x = torch.randn(2, 30, 48, device="cuda")
    announce("GatedFeedForward")
    a = x.double().cpu().numpy().reshape(60, 48)
    h = reference(torch.tensor(a), m.gate_proj.weight, m.up_proj.weight, None, None, "gelu")
    check(m(x).reshape(60, 48), h @ m.down_proj.weight.detach().double().cpu().numpy().T, torch.float32, "block")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = G.gated_linear(x, m.gate_proj.weight, m.up_proj.weight, activation="gelu")
        assert y.dtype == torch.bfloat16
        y.float().sum().backward()
    assert m.gate_proj.weight.grad.dtype == torch.float32


def test_refusals(G):
    x, w = torch.zeros(2, 8, device="cuda"), torch.zeros(5, 8, device="cuda")
    b = torch.zeros(5, device="cuda")
    for match, args in (("one dtype on one GPU", (x.half(), w.half(), w.half())), ("one dtype", (x, w.bfloat16(), w)),
                        ("one dtype", (x.cpu(), w, w)), ("one dtype", (x, w, w, b.cpu())),
                        ("expected x", (x[:, :7], w, w)), ("expected x", (x, w, w[:4])), ("expected x", (x, w[0], w)),
                        ("expected x", (x, w, w, b[:4]))):
        with pytest.raises(RuntimeError, match=match):
            G.gated_linear(*args)
    with pytest.raises(ValueError, match="activation must be one of"):
        G.gated_linear(x, w, w, activation="tanh")
    with pytest.raises(ValueError, match="activation must be one of"):
        G.GatedFeedForward(8, 8, activation="swish")
    wide = torch.zeros(2, 2 ** 20 + 8, device="cuda")
    with pytest.raises(RuntimeError, match="row strides up to"):
        G.gated_linear(wide, wide, wide)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_single_columns_of_any_row_stride(G, dtype):
    """One column broadcast from one row (a summed loss's gradient, an expanded input or
    weight), or of a matrix whose rows lie further apart than the kernels take."""
    far = (1 << 20) + 8
    for T, D, n in ((9, 24, 1), (70, 1, 50), (700, 1, 1), (3, 1, 200)):
        args, _ = inputs(T, D, n, dtype, True, seed=T)
        cases = [("dense", args)]
        if D == 1:
            cases.append(("expanded", [args[0][:1].expand(T, 1), *(w[:1].expand(n, 1) for w in args[1:3]), *args[3:]]))
        if D == 1 and T <= 70:
            wide = torch.empty(T, far, dtype=dtype, device="cuda")
            wide[:, :1] = args[0]
            cases.append(("far apart", [wide[:, :1], *args[1:]]))
        for name, given in cases:
            announce(f"gated_linear single columns {(T, D, n)} {dtype} {name}")
            want = reference(*given, "gelu", torch.ones(T, n))
            with torch.no_grad():
                check(G.gated_linear(*given, activation="gelu"), want[0], dtype, f"{name} y")
            leaves = [t.detach().requires_grad_(True) for t in given]
            y = G.gated_linear(*leaves, activation="gelu")
            for g, w, what in zip(torch.autograd.grad(y.sum(), leaves), want[1:], ("x", "gate", "up", "gate bias", "up bias")):
                check(g, w, dtype, f"{name} grad {what}", True)


def test_shared_inputs_differentiate_twice(G):
    """create_graph where gate and up share a weight and a bias, and where a block is applied
    twice: gradients and second derivatives as float64's of the separate steps."""
    args, _ = inputs(20, 24, 24, torch.float32, True, seed=10, scale=1.0)
    x, w, v, b, c = (t * 0.5 for t in args)
    tied = lambda f, x, w, b: f(x, w, w, b, b)  # noqa: E731
    twice = lambda f, x, w, v, b, c: f(f(x, w, v, b, c), w, v, b, c)  # noqa: E731
    for name, use, given in (("tied", tied, (x, w, b)), ("twice", twice, (x, w, v, b, c))):
        announce(f"gated_linear create_graph {name}")
        seen = []
        for cast, f in ((torch.Tensor.cuda, G.gated_linear), (lambda t: t.double().cpu(), lambda *a: G._separate(*a, "silu"))):
            leaves = [cast(t.detach()).clone().requires_grad_(True) for t in given]
            grads = torch.autograd.grad(use(f, *leaves).square().sum(), leaves, create_graph=True)
            seen.append((*grads, *torch.autograd.grad(sum(t.square().sum() for t in grads), leaves)))
        for got, want in zip(*seen):
            # the float32 steps of two blocks and three derivatives, sums of at most 24 x 20 terms
            assert torch.allclose(got.double().cpu(), want, rtol=1e-4, atol=1e-4 * float(want.abs().max())), name


def test_forward_mode_is_refused(G):
    """A tangent raises, whichever argument carries it, under no_grad too."""
    from torch.autograd import forward_ad

    args, _ = inputs(5, 8, 6, torch.float32, True)
    announce("gated_linear with tangents")
    with forward_ad.dual_level():
        G.gated_linear(*args)
        for i, t in enumerate(args):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else u for j, u in enumerate(args)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                G.gated_linear(*dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                G.gated_linear(*dual)


@torch.random.fork_rng()  # later tests draw what they drew
@pytest.mark.parametrize("which", ["gate_proj", "up_proj"])
def test_module_runs_replaced_and_hooked_projections(G, which):
    """A projection that is more than its weight and bias is called as it is."""
    torch.manual_seed(1)
    m = G.GatedFeedForward(20, 36, bias=True).cuda()
    x = torch.randn(7, 20, device="cuda")
    getattr(m, which).register_forward_hook(lambda mod, args, out: 2 * out + 1)
    announce(f"GatedFeedForward with a hook on {which}")
    want = m.down_proj(torch.nn.functional.silu(m.gate_proj(x)) * m.up_proj(x))
    assert torch.allclose(m(x), want, rtol=1e-5, atol=1e-5 * float(want.detach().abs().max()))
    setattr(m, which, torch.nn.Sequential(torch.nn.Linear(20, 36), torch.nn.Dropout(0.0)).cuda())
    want = m.down_proj(torch.nn.functional.silu(m.gate_proj(x)) * m.up_proj(x))
    assert torch.allclose(m(x), want, rtol=1e-5, atol=1e-5 * float(want.detach().abs().max()))
    setattr(m, which, torch.nn.utils.parametrizations.weight_norm(torch.nn.Linear(20, 36)).cuda())
    want = m.down_proj(torch.nn.functional.silu(m.gate_proj(x)) * m.up_proj(x))
    assert torch.allclose(m(x), want, rtol=1e-5, atol=1e-5 * float(want.detach().abs().max()))


def test_empty_batch_of_large_weights(G):
    """Zeros for more of a weight's gradient than a launch has threads for, two bytes each."""
    from ossm_amd import _lib

    n, D = 1 << 19, 4100
    grad = torch.ones(n, D, device="cuda")
    assert grad.numel() * 4 > 2 ** 33
    announce("gated_linear backward of an empty batch, 8.6 GB of weights")
    _lib.run(_lib.load().ossm_gated_backward, grad, 0, None, n, None, D, None, D, None, D, 0, None, None, None,
             grad.data_ptr(), None, None, None, 0, D, n)
    assert not grad.any()
