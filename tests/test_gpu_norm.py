"""GPU tests of layer norm (ossm_amd.norm), forward and backward, against float64
formulas, and of its gradients against differences.

Tolerances, derived before the first run, u = 2^-24.  A row's mean is a sum in which an
element passes at most 48 roundings (32 of a lane's, 10 of the lanes' and waves'), so it is off by
48 u max|s| at most, n = (s - mean) rstd by dn = u (48 max|s| rstd + 16 |n|), the
last term for the variance's and the root's roundings; y = n w + b by dn |w| + 4 u (|n w| + |b|).
ds = rstd (g - mean(g) - n mean(g n)): each term's own roundings, 16 u of it, the means' 48 u of
the means of |g| and |g n|, and dn times |mean(g n)| and, inside that mean, |n| times the
mean of |g| dn.  dw = sum gy n: dn |gy| of each row and (rows + 24) u of the sum of |gy n|.  The
result's rounding is finfo.eps / 2 of it, to bfloat16 2^-8."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]
NAMES = ["f32", "bf16", "bf16-f32"]


@pytest.fixture(scope="module")
def N():
    need_gpu()
    from ossm_amd import norm

    return norm


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def rounded(a, dtype):
    return torch.tensor(a).to(dtype).double().numpy()


def reference(x, res, w, b, gy=None, gs=None, eps=EPS):
    """Results and tolerances without the results' own rounding: y, s, ds, dw, db."""
    dtype = x.dtype
    x, res, w, b, gy, gs = map(f64, (x, res, w, b, gy, gs))
    s = x if res is None else rounded(x + res, dtype)
    w = np.ones(s.shape[1]) if w is None else w
    b = np.zeros(s.shape[1]) if b is None else b
    mean = s.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((s - mean) ** 2).mean(1, keepdims=True) + eps)
    n = (s - mean) * rstd
    dn = U * (48 * np.abs(s).max(1, keepdims=True) * rstd + 16 * np.abs(n))
    out = {"y": (n * w + b, dn * np.abs(w) + 4 * U * (np.abs(n * w) + np.abs(b))), "s": (s, 0 * s)}
    if gy is None:
        return out
    g = gy * w
    m1, m2 = g.mean(1, keepdims=True), (g * n).mean(1, keepdims=True)
    a1, a2 = np.abs(g).mean(1, keepdims=True), np.abs(g * n).mean(1, keepdims=True)
    ds = rstd * (g - m1 - n * m2)
    tol = rstd * (U * (16 * (np.abs(g) + np.abs(m1) + np.abs(n * m2)) + 64 * (a1 + np.abs(n) * a2))
                  + dn * np.abs(m2) + np.abs(n) * (np.abs(g) * dn).mean(1, keepdims=True))
    if gs is not None:
        ds, tol = ds + gs, tol + 2 * U * np.abs(ds + gs)
    rows = len(s) + 24
    out["ds"] = ds, tol
    out["dw"] = (gy * n).sum(0), (np.abs(gy) * dn).sum(0) + rows * U * np.abs(gy * n).sum(0)
    out["db"] = gy.sum(0), rows * U * np.abs(gy).sum(0)
    return out


def check(got, want, what):
    value, tol = want
    g = f64(got)
    assert g.shape == value.shape, what
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(g - value) <= tol + torch.finfo(got.dtype).eps / 2 * np.abs(value) + 1e-37) |
                (np.isnan(g) & np.isnan(value)))
    assert not bad.any(), f"{what}: {int(bad.sum())}/{bad.size} off, first at {np.argwhere(bad)[0]}"


def inputs(T, D, dtype, wdtype, residual, seed=0, shift=0.5):
    rng = np.random.default_rng(seed)
    f = lambda *s, k=1.0, c=0.0, t=dtype: torch.tensor(rng.normal(size=s) * k + c).to(t).cuda()  # noqa: E731
    return (f(T, D), f(T, D, k=3, c=shift) if residual else None, f(D, k=0.3, c=1, t=wdtype), f(D, t=wdtype), f(T, D),
            f(T, D) if residual else None)


def run(N, x, res, w, b, gy, gs, eps=EPS):
    leaves = [t if t is None else t.detach().requires_grad_(True) for t in (x, res, w, b)]
    lx, lr, lw, lb = leaves
    if res is None:
        y, s = N.layer_norm(lx, lw, lb, eps), None
        outs, grads = [y], [gy]
    else:
        y, s = N.add_layer_norm(lx, lr, lw, lb, eps)
        outs, grads = [y, s], [gy, gs]
    got = iter(torch.autograd.grad(outs, [t for t in leaves if t is not None], grads))
    return y.detach(), None if s is None else s.detach(), [None if t is None else next(got) for t in leaves]


SIZES = [(1, 1), (3, 2), (5, 7), (2, 8), (9, 31), (33, 32), (17, 33), (70, 64), (6, 65), (40, 128), (11, 129), (3, 256), (2, 257),
         (5, 511), (4, 513), (300, 1022), (7, 1025), (3, 2047), (4, 2048), (2, 2049), (3, 4097), (2, 8191), (2, 8200),
         (2, 16384), (2, 16385), (3, 40001), (1, 2048), (5000, 24)]


@pytest.mark.parametrize("types", TYPES, ids=NAMES)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_matches_float64(N, size, types):
    T, D = size
    dtype, wdtype = types
    for residual in (False, True):
        x, res, w, b, gy, gs = inputs(T, D, dtype, wdtype, residual, seed=D)
        want = reference(x, res, w, b, gy, gs)
        announce(f"layer norm {size} {types} residual {residual}")
        with torch.no_grad():
            if residual:
                y0, s0 = N.add_layer_norm(x, res, w, b)
            else:
                y0, s0 = N.layer_norm(x, w, b), None
        y, s, (dx, dres, dw, db) = run(N, x, res, w, b, gy, gs)
        assert torch.equal(y, y0) and y.dtype == dtype
        check(y, want["y"], "y")
        check(dx, want["ds"], "dx")
        check(dw, want["dw"], "dw")
        check(db, want["db"], "db")
        assert dw.dtype == wdtype
        if residual:
            assert torch.equal(s, s0) and torch.equal(dx, dres)
            check(s, want["s"], "s")
        again = run(N, x, res, w, b, gy, gs)
        assert torch.equal(again[2][2], dw) and torch.equal(again[2][0], dx)  # bitwise


def test_far_from_zero_and_constant_rows(N):
    """The variance is about the mean: a mean of a thousand deviations costs its own digits
    only.  A constant row has no variance: y is the bias."""
    x, _, w, b, gy, _ = inputs(6, 700, torch.float32, torch.float32, False, seed=1)
    x += 1000.0
    x[2] = 7.0
    announce("layer norm far from zero")
    want = reference(x, None, w, b, gy)
    y, _, (dx, _, dw, db) = run(N, x, None, w, b, gy, None)
    check(y, want["y"], "y")
    check(dx, want["ds"], "dx")
    check(dw, want["dw"], "dw")
    assert torch.equal(y[2], b)


def test_gradients_of_equal_elements(N):
    """With every element equal, nothing but the sum's own gradient is left of a row where the
    gradients times the weights are equal too: their mean is exact at 1, 2 and 64 columns (sums of equal
    numbers by pairs), and at 3 off by at most 2 U of it, which rstd = eps^-1/2 carries."""
    for D in (1, 2, 3, 64):
        for dtype in (torch.float32, torch.bfloat16):
            announce(f"norm of equal elements {D} {dtype}")
            rng = np.random.default_rng(D)
            one = lambda *shape: torch.tensor(rng.normal(size=shape)).to(dtype).cuda()  # noqa: E731
            x, gy, gs = one(500, 1).repeat(1, D), one(500, 1).repeat(1, D), one(500, D)
            res = torch.zeros_like(x)
            w, b = one(1).float().repeat(D), one(D).float()
            leaves = [t.requires_grad_(True) for t in (x, res, w, b)]
            y, s = N.add_layer_norm(*leaves)
            got = torch.autograd.grad([y, s], leaves[:2], [gy, gs])
            most = 0.0 if D != 3 else 2 * U * EPS ** -0.5 * float((gy.float() * w.detach()).abs().max())
            for g in got:
                off = (g.double() - gs.double()).abs()
                assert bool((off <= most * (1 + 2 * U) + (0 if D != 3 else torch.finfo(dtype).eps / 2) * (gs.double().abs() + most)).all()), (D, dtype, float(off.max()))


def test_rows_do_not_reach_one_another(N):
    """A row with NaN or infinities gives NaN, the others what they give alone."""
    for D in (24, 128, 2048, 5000, 20000):
        x, res, w, b, gy, gs = inputs(9, D, torch.float32, torch.float32, True, seed=2)
        clean = run(N, x, res, w, b, gy, gs)
        x[3, 1], x[5, 0], res[7, D - 1] = float("nan"), float("inf"), -float("inf")
        announce(f"layer norm special values {D}")
        y, s, (dx, _, dw, db) = run(N, x, res, w, b, gy, gs)
        for r in range(9):
            if r in (3, 5, 7):
                assert torch.isnan(y[r]).any() and torch.isnan(dx[r]).any()
            else:
                assert torch.equal(y[r], clean[0][r]) and torch.equal(dx[r], clean[2][0][r])
        assert torch.isnan(dw).any() and torch.equal(db, clean[2][3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides_offsets_and_other_streams(N, dtype):
    """Rows at every offset, wide strides, broadcast rows and gradients, another stream: all
    what dense tensors give."""
    T, D = 5, 1021
    x, res, w, b, gy, gs = inputs(T, D, dtype, dtype, True, seed=3)
    want = run(N, x, res, w, b, gy, gs)
    for off in range(1, 9):
        wide = lambda t: torch.zeros(T, D + 40, dtype=dtype, device="cuda")[:, off:off + D].copy_(t)  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        announce(f"layer norm offset {off} {dtype}")
        with torch.cuda.stream(side):
            got = run(N, *(wide(t) for t in (x, res)), w, b, wide(gy), wide(gs))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert all(torch.equal(p, q) for p, q in zip(got[2], want[2]))
    announce("layer norm of transposed, broadcast and three-dimensional tensors")
    got = run(N, x.t().contiguous().t(), res, w, b, gy, gs)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2][0], want[2][0])
    one = x[:1].expand(T, D)
    assert torch.equal(N.layer_norm(one, w, b), N.layer_norm(one.contiguous(), w, b))
    ones = torch.ones(1, 1, dtype=dtype, device="cuda").expand(T, D)
    leaf = x.clone().requires_grad_(True)
    g1, = torch.autograd.grad(N.layer_norm(leaf, w, b).sum(), leaf)
    g2, = torch.autograd.grad(N.layer_norm(leaf, w, b), leaf, ones.contiguous())
    assert torch.equal(g1, g2)
    cube = x[:4].view(2, 2, D)
    y, s = N.add_layer_norm(cube, res[:4].view(2, 2, D), w, b)
    assert y.shape == cube.shape and torch.equal(s.view(4, D), want[1][:4]) and torch.equal(y.view(4, D), want[0][:4])
    assert torch.equal(N.layer_norm(x[0], w, b), N.layer_norm(x[:1], w, b)[0])


def test_parts_alone(N):
    """No weight, no bias, one of them; gradients of some inputs only, of one output only."""
    x, res, w, b, gy, gs = inputs(12, 200, torch.float32, torch.float32, True, seed=4)
    announce("layer norm parts alone")
    for pw, pb in ((None, None), (w, None), (None, b)):
        want = reference(x, res, pw, pb, gy, gs)
        y, s, (dx, _, dw, db) = run(N, x, res, pw, pb, gy, gs)
        check(y, want["y"], "y")
        check(dx, want["ds"], "dx")
        if pw is not None:
            check(dw, want["dw"], "dw")
        if pb is not None:
            check(db, want["db"], "db")
    want = reference(x, res, w, b, gy, None)
    lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y, s = N.add_layer_norm(lx, res, lw, b)
    dx, = torch.autograd.grad(y, lx, gy, retain_graph=True)
    check(dx, want["ds"], "dx of y alone")
    dw, = torch.autograd.grad(y, lw, gy, retain_graph=True)
    check(dw, want["dw"], "dw alone")
    dx, dw = torch.autograd.grad(s, [lx, lw], gs, retain_graph=True, allow_unused=True)
    assert torch.equal(dx, gs) and (dw is None or not dw.any())
    # the same tensor as both terms: its gradients add up
    both = x.clone().requires_grad_(True)
    y, s = N.add_layer_norm(both, both, w, b)
    d, = torch.autograd.grad([y, s], both, [gy, gs])
    check(d, tuple(2 * t for t in reference(x, x, w, b, gy, gs)["ds"]), "a tensor given twice")


def test_against_differences(N):
    """Gradients against central differences of the kernel's own outputs: of a loss of some
    size 1, with a step of 2^-7 the difference's error is u / step + step^2 of its terms, below 2e-3."""
    x, res, w, b, gy, gs = inputs(3, 37, torch.float32, torch.float32, True, seed=5)
    _, _, grads = run(N, x, res, w, b, gy, gs)

    def loss(*t):
        y, s = N.add_layer_norm(*t)
        return (y.double() * gy.double()).sum().item() + (s.double() * gs.double()).sum().item()

    announce("layer norm against differences")
    rng = np.random.default_rng(0)
    args = [x, res, w, b]
    for k, (t, g) in enumerate(zip(args, grads)):
        d = torch.tensor(rng.normal(size=t.shape)).float().cuda()
        h = 2.0 ** -7
        up, down = (loss(*(a + sign * h * d if i == k else a for i, a in enumerate(args))) for sign in (1, -1))
        along = (g.double() * d.double()).sum().item()
        size = (g.double() * d.double()).abs().sum().item()
        assert abs((up - down) / (2 * h) - along) <= 2e-3 * size + 2e-3, k


def test_second_derivatives(N):
    """create_graph differentiates as the separate steps, a tensor that enters twice too."""
    x, res, w, b, gy, gs = (t.double().float() for t in inputs(4, 19, torch.float32, torch.float32, True, seed=6))

    def second(norm):
        leaves = [t.clone().requires_grad_(True) for t in (x, res, w, b)]
        h = leaves[0] * 2
        y, s = norm(h, leaves[1] + h, leaves[2], leaves[3])
        g = torch.autograd.grad([y, s], leaves, [gy, gs], create_graph=True)
        return torch.autograd.grad(sum((t * t).sum() for t in g), leaves, allow_unused=True)

    def plain(p, q, w_, b_):
        s = p + q
        return torch.nn.functional.layer_norm(s, s.shape[-1:], w_, b_), s

    announce("layer norm second derivatives")
    for got, want in zip(second(N.add_layer_norm), second(plain)):
        if want is None:
            assert got is None or not got.any()
        else:
            assert (got - want).abs().max() <= 1e-4 * want.abs().max()


def test_empty_and_long_batches(N):
    w = torch.ones(5).cuda()
    announce("layer norm of nothing")
    x = torch.zeros(0, 5).cuda().requires_grad_(True)
    lw = w.clone().requires_grad_(True)
    y = N.layer_norm(x, lw, w)
    dx, dw = torch.autograd.grad(y, [x, lw], torch.zeros_like(y))
    assert y.shape == (0, 5) and dx.shape == (0, 5) and not dw.any()
    assert N.layer_norm(torch.zeros(3, 0).cuda()).shape == (3, 0)
    y, s = N.add_layer_norm(torch.zeros(2, 0, 5).cuda(), torch.zeros(2, 0, 5).cuda(), w, w)
    assert y.shape == s.shape == (2, 0, 5)


def test_past_32_bits(N):
    """Rows that start past 2^31 elements, forward and backward."""
    D = 2048
    T = 2 ** 20 + 5
    x = torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    x.view(-1)[:] = 1.0
    some = torch.randn(5, D, device="cuda").bfloat16()
    x[-5:] = some
    w, b = torch.randn(D).cuda().bfloat16(), torch.randn(D).cuda().bfloat16()
    announce("layer norm past 2^31 elements")
    y = N.layer_norm(x, w, b)
    assert torch.equal(y[-5:], N.layer_norm(some, w, b))
    leaf = x.requires_grad_(True)
    d, = torch.autograd.grad(N.layer_norm(leaf, w, b), leaf, y)
    want = run(N, some, None, w, b, y[-5:], None)[2][0]
    assert torch.equal(d[-5:], want)


def test_graph_capture(N):
    """Forward and backward in a captured graph, replayed on changing inputs between eager
    calls, each replay against the eager result."""
    x, res, w, b, gy, gs = inputs(50, 300, torch.float32, torch.float32, True, seed=7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(N, x, res, w, b, gy, gs)
    torch.cuda.synchronize()
    announce("layer norm under graph capture")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, s, grads = run(N, x, res, w, b, gy, gs)
    for i in range(4):
        x.normal_()
        gy.normal_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        want = run(N, x, res, w, b, gy, gs)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(s, want[1]), f"replay {i}"
        assert all(torch.equal(p, q) for p, q in zip(grads, want[2])), f"replay {i}"


def test_module_and_autocast(N):
    m = N.LayerNorm(96).cuda()
    torch.nn.init.normal_(m.weight)
    plain = torch.nn.LayerNorm(96).cuda()
    plain.load_state_dict(m.state_dict())
    x = torch.randn(4, 7, 96).cuda()
    announce("LayerNorm module")
    assert (m(x) - plain(x)).abs().max() <= 1e-5
    y, s = m(x, x)
    assert torch.equal(s, 2 * x) and (y - plain(2 * x)).abs().max() <= 1e-5
    with torch.autocast("cuda", torch.bfloat16):
        y, s = m(x.bfloat16(), x)
        want = plain(x.bfloat16() + x)
        assert y.dtype == want.dtype == torch.float32 and (y - want).abs().max() <= 1e-5
    with pytest.raises(RuntimeError, match="last dimension"):
        m(x[..., :5])
    with pytest.raises(RuntimeError, match="last dimension"):
        N.LayerNorm((7, 96)).cuda()(x)


def test_refusals(N):
    x, w = torch.zeros(3, 8).cuda(), torch.ones(8).cuda()
    for match, args in (("x must be", (x.half(), None, None)), ("x must be", (x.cpu(), None, None)),
                        ("x must be", (x[0, 0], None, None)), ("weight and bias", (x, w[:4], None)),
                        ("weight and bias", (x, w.double(), None)), ("weight and bias", (x, w.bfloat16(), None)),
                        ("weight and bias", (x.bfloat16(), w, w.bfloat16())), ("weight and bias", (x, w, w.cpu()))):
        with pytest.raises(RuntimeError, match=match):
            N.layer_norm(*args)
    for res in (x[:2], x.bfloat16(), x.cpu()):
        with pytest.raises(RuntimeError, match="residual must be"):
            N.add_layer_norm(x, res, w, w)
    from torch.autograd import forward_ad

    announce("layer norm with tangents")
    with torch.no_grad(), forward_ad.dual_level(), pytest.raises(RuntimeError, match="tangent"):
        N.layer_norm(forward_ad.make_dual(x, torch.ones_like(x)), w, w)


def test_float32_rows_of_equal_large_elements(N):
    """A constant row's deviations are all zero, whatever its value and length: y is the bias and
    the gradient's factor is eps^-1/2.  ds = rstd (g - mean(g)) then, each term's roundings 16 U of it and
    the mean's 64 U of the mean of |g|, as in `reference`."""
    rng = np.random.default_rng(20)
    for D in (3, 23, 100, 701, 7879, 15237, 40001):
        T = 64
        value = torch.tensor(np.exp(rng.uniform(np.log(1e3), np.log(1e11), size=(T, 1)))).float()
        x = value.repeat(1, D).cuda()
        half = (value / 2).repeat(1, D).cuda()  # exact: its double is the value
        _, _, w, b, gy, gs = inputs(T, D, torch.float32, torch.float32, True, seed=D)
        for eps in (1e-5, 1e-12):
            announce(f"layer norm of equal large elements {D} {eps}")
            y, _, (dx, _, dw, db) = run(N, x, None, w, b, gy, None, eps)
            assert torch.equal(y, b.expand(T, D)), (D, eps, float((y - b).abs().max()))
            g = f64(gy) * f64(w)
            m1, a1 = g.mean(1, keepdims=True), np.abs(g).mean(1, keepdims=True)
            root = np.float32(eps) ** np.float64(-0.5)
            check(dx, (root * (g - m1), root * U * (16 * (np.abs(g) + np.abs(m1)) + 64 * a1)), "dx")
            assert not dw.any()
            y, s, _ = run(N, half, half, w, b, gy, gs, eps)
            assert torch.equal(y, b.expand(T, D)) and torch.equal(s, x)


def test_float32_rows_of_nearly_equal_large_elements(N):
    """Elements a few units in the last place apart: their differences are exact, so the deviations
    keep their digits.  A mean of differences of up to 5 units is off by 48 U of 5 units, and a
    deviation's own rounding and the root's are 16 U of n, as in the module's derivation with the largest
    difference in place of the largest element."""
    rng = np.random.default_rng(21)
    for D in (33, 701, 7879, 15237, 40001):
        T = 24
        base = np.float32(2.0) ** rng.integers(10, 36, size=(T, 1))
        unit = base * 2.0 ** -23
        x = torch.tensor(base * 1.5 + unit * rng.integers(-2, 4, size=(T, D))).float().cuda()
        _, _, w, b, _, _ = inputs(T, D, torch.float32, torch.float32, False, seed=D)
        announce(f"layer norm of nearly equal large elements {D}")
        y = N.layer_norm(x, w, b, 1e-12)
        s, w64, b64 = f64(x), f64(w), f64(b)
        c = s - s.mean(1, keepdims=True)
        rstd = 1 / np.sqrt((c ** 2).mean(1, keepdims=True) + float(np.float32(1e-12)))
        n = c * rstd
        dn = U * (48 * 5 * unit * rstd + 16 * np.abs(n))
        check(y, (n * w64 + b64, dn * np.abs(w64) + 4 * U * (np.abs(n * w64) + np.abs(b64))), "y")


def test_the_sum_alone_is_not_reached_by_the_norm(N):
    """A loss of the sum alone: its gradient is the sum's own, also in rows whose norm is NaN, and
    the weights get none."""
    x, res, w, b, _, gs = inputs(4, 40, torch.float32, torch.float32, True, seed=22)
    x[1, 3], x[2, 0] = float("inf"), float("nan")
    announce("layer norm, the sum alone")
    for graph in (False, True):
        leaves = [t.clone().requires_grad_(True) for t in (x, res, w, b)]
        _, s = N.add_layer_norm(*leaves)
        dx, dres, dw, db = torch.autograd.grad(s, leaves, gs, allow_unused=True, create_graph=graph)
        assert torch.equal(dx, gs) and torch.equal(dres, gs) and dw is None and db is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_training_on_tensors_of_any_shape(N, dtype):
    """Dense, transposed, cut out and broadcast tensors and gradients of one to four dimensions: what
    their matrices give, outputs dense."""
    D = 37
    _, _, w, b, _, _ = inputs(1, D, dtype, torch.float32, False, seed=23)
    rand = lambda *s: torch.randn(*s, device="cuda").to(dtype)  # noqa: E731
    with torch.random.fork_rng():
        torch.manual_seed(5)
        cases = [[rand(D) for _ in range(4)], [rand(2, 3, D) for _ in range(4)], [rand(2, 1, 3, D) for _ in range(4)],
                 [rand(3, 2, D).transpose(0, 1) for _ in range(4)], [rand(2, 5, D)[:, 1:4] for _ in range(4)],
                 [rand(2, D, 3).transpose(1, 2) for _ in range(4)], [rand(2, 3, 2 * D)[..., ::2] for _ in range(4)],
                 [rand(1, 1, D).expand(2, 3, D) for _ in range(4)], [rand(2, 3, 1).expand(2, 3, D) for _ in range(4)],
                 [rand(2, 0, D) for _ in range(4)], [rand(5, 1, D).as_strided((5, 1, D), (D, 10 ** 6, 1)) for _ in range(4)]]
    for x, res, gy, gs in cases:
        announce(f"layer norm training {tuple(x.shape)} {x.stride()}")
        flat = [t.reshape(-1, D).contiguous() for t in (x, res, gy, gs)]
        for two in (False, True):
            y, s, grads = run(N, x, res if two else None, w, b, gy, gs)
            wy, ws, want = run(N, flat[0], flat[1] if two else None, w, b, *flat[2:])
            assert y.shape == x.shape and y.is_contiguous() and torch.equal(y.view(-1, D), wy)
            assert not two or s.shape == x.shape and torch.equal(s.view(-1, D), ws)
            for p, q in zip(grads, want):
                assert (p is None and q is None) or torch.equal(p.reshape(q.shape), q)
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, res)]
        y, s = N.add_layer_norm(*leaves, w, b)
        g1 = torch.autograd.grad([y, s], leaves, [gy, gs], create_graph=True)
        g2 = torch.autograd.grad([y, s], leaves, [gy, gs])
        for p, q in zip(g1, g2):
            assert p.shape == q.shape == x.shape
            assert x.numel() == 0 or (p - q).abs().max() <= (1e-4 if dtype == torch.float32 else 0.05) * q.abs().max()
