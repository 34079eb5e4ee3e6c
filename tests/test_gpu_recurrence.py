"""GPU tests of the gated linear recurrence (ossm_amd.recurrence): training forward and
backward, packed prompts and single tokens, against float64 loops over time, and the
gradients against differences.

Tolerances, derived before the first run, u = 2^-24.  A sigmoid is off by at most 6 u of itself
(an exponential of 3, a sum, a reciprocal), so l = -k sigmoid(r) by 10 u (k: 3, a product), a by
(10 |l| + 4) u a.  m = sqrt(1 - a^2) moves by half of l's relative error where |l| is small, and where it
comes from a itself (a^2 < 0.67) by a^2 / (1 - a^2) <= 2 times a's relative error at |l| <= 0.2 and less
beyond, at most 14 u m; the step's input b = m g x thus by 24 u |b|.  The state's error runs along:
  e_t = a_t (e_{t-1} + (10 |l| + 6) u |h_{t-1}|) + 26 u |b_t|
where joining chunks multiplies by exp of sums of l, whose errors are the sums of theirs, and six
more roundings a joint (a chunk is at least 8 steps): u (|h| / 1) a step bounds those.  The gradient's error runs
backwards the same way, E_t; a product's relative errors add up.  1 - sigmoid loses 6 u of one.
Where |l| is below float32's smallest normal number, 2^-126, it may be lost, and with it m = sqrt(2 |l|) and
-l / m = sqrt(|l| / 2) up to M0 = 2^-62 (2^-62.5 and 2^-63.5): M0 of the factors that stand beside them.
The results' rounding is finfo.eps / 2, to bfloat16 2^-8."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.gpu_util import announce, need_gpu, no_device_errors

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
M0 = 2.0 ** -62


@pytest.fixture(scope="module")
def R():
    need_gpu()
    from ossm_amd import recurrence

    return recurrence


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def sig(v):
    return 1 / (1 + np.exp(-v))


def softplus(v):
    return np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))


class Parts:
    """A step's values, all steps at once."""

    def __init__(self, x, i, r, z, decay, scale):
        self.x, self.g, self.open = x, sig(i), sig(r)
        self.l = -scale * softplus(decay) * self.open
        self.a = np.exp(self.l)
        self.m = np.sqrt(-np.expm1(2 * self.l))
        self.b = self.m * self.g * x
        self.z = z
        self.out = np.ones_like(x) if z is None else z * sig(z)


def scan(p, start, axis_len):
    """States [B, L, D], their errors, from start; p's arrays [B, L, D]."""
    h, e = start.copy(), np.zeros_like(start)
    hs, es = [], []
    for t in range(axis_len):
        a = p.a[:, t]
        e = a * (e + (10 * np.abs(p.l[:, t]) + 7) * U * np.abs(h)) + 26 * U * np.abs(p.b[:, t]) + M0 * np.abs(p.x[:, t])
        h = a * h + p.b[:, t]
        hs.append(h)
        es.append(e)
    return np.stack(hs, 1), np.stack(es, 1)


def reference(x, i, r, z, decay, start, scale, gy=None, glast=None):
    """{name: (value, tolerance before the result's own rounding)}."""
    x, i, r, z, decay, start, gy, glast = map(f64, (x, i, r, z, decay, start, gy, glast))
    B, L, D = x.shape
    p = Parts(x, i, r, z, decay, scale)
    h0 = np.zeros((B, D)) if start is None else start
    h, e = scan(p, h0, L)
    y = h * p.out
    out = {"y": (y, e * np.abs(p.out) + 10 * U * np.abs(y)), "last": (h[:, -1], e[:, -1])}
    if gy is None:
        return out
    go = gy * p.out
    G, E = np.zeros_like(x), np.zeros_like(x)
    g = np.zeros((B, D)) if glast is None else glast
    err = np.zeros((B, D))
    for t in range(L - 1, -1, -1):
        err = err + 12 * U * np.abs(go[:, t])
        g = g + go[:, t]
        G[:, t], E[:, t] = g, err
        err = p.a[:, t] * (err + (10 * np.abs(p.l[:, t]) + 7) * U * np.abs(g))
        g = p.a[:, t] * g
    out["start"] = g, err
    before, eb = np.concatenate([h0[:, None], h[:, :-1]], 1), np.concatenate([0 * h0[:, None], e[:, :-1]], 1)
    gm = G * p.m * p.g
    out["x"] = gm, E * p.m * p.g + 24 * U * np.abs(gm) + M0 * np.abs(G)
    gi = gm * x * (1 - p.g)
    out["i"] = gi, E * np.abs(p.m * p.g * x * (1 - p.g)) + 30 * U * np.abs(gi) + 6 * U * np.abs(gm * x) + M0 * np.abs(G * x)
    back = np.where(p.m > 0, p.a ** 2 * -p.l / np.where(p.m > 0, p.m, 1), 0)
    q1, q2 = p.a * p.l * before, p.g * x * back
    q = G * (q1 + q2)
    tq = E * np.abs(q1 + q2) + np.abs(G) * (np.abs(p.a * p.l) * eb + (20 * np.abs(p.l) + 50) * U * (np.abs(q1) + np.abs(q2))
                                           + M0 * np.abs(x))
    gr = q * (1 - p.open)
    out["r"] = gr, tq * (1 - p.open) + 30 * U * np.abs(gr) + 6 * U * np.abs(q)
    ratio = sig(decay) / softplus(decay)
    gd = ratio * q.sum((0, 1))
    out["decay"] = gd, ratio * (tq.sum((0, 1)) + 30 * U * np.abs(q).sum((0, 1))) + 8 * U * np.abs(gd)
    if z is not None:
        s = sig(z)
        gz = gy * h * s * (1 + z * (1 - s))
        out["z"] = gz, np.abs(gy) * s * (1 + np.abs(z)) * (e + 20 * U * np.abs(h))
    return out


def check(got, want, what):
    value, tol = want
    g = f64(got)
    assert g.shape == value.shape, what
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(g - value) <= tol + torch.finfo(got.dtype).eps / 2 * np.abs(value) + 1e-36)
    assert not bad.any(), (f"{what}: {int(bad.sum())}/{bad.size} off, worst {np.max(np.abs(g - value) / (tol + 1e-36)):.1f} of the "
                           f"tolerance, first at {np.argwhere(bad)[0]}")


def inputs(B, L, D, dtype, gate, state, seed=0, spread=1.0):
    rng = np.random.default_rng(seed)
    f = lambda *s, k=1.0, t=dtype: torch.tensor(rng.normal(size=s) * k).to(t).cuda()  # noqa: E731
    rate = np.exp(rng.uniform(np.log(5e-4), np.log(0.5), D))
    decay = torch.tensor(np.log(np.expm1(2 * rate / 8))).float().cuda()
    x, i, r, z = f(B, L, D), f(B, L, D, k=spread), f(B, L, D, k=spread), f(B, L, D) if gate else None
    return [x, i, r, z, decay, f(B, D, t=torch.float32) if state else None], f(B, L, D), f(B, D, t=torch.float32)


NAMES = ("x", "i", "r", "z", "decay", "start")


def train(R, x, i, r, z, decay, start, scale=8.0):
    return R.gated_recurrence(x, i, r, decay, z, start, scale=scale)


def run(R, args, gy, glast, scale=8.0, wanted=NAMES):
    leaves = [t if t is None else t.detach().requires_grad_(n in wanted) for n, t in zip(NAMES, args)]
    y, last = train(R, *leaves, scale)
    outs = [(o, g) for o, g in ((y, gy), (last, glast)) if g is not None]
    need = {n: t for n, t in zip(NAMES, leaves) if t is not None and n in wanted}
    grads = torch.autograd.grad([o for o, _ in outs], list(need.values()), [g for _, g in outs])
    return {"y": y.detach(), "last": last.detach(), **dict(zip(need, grads))}


SIZES = [(1, 1, 1), (2, 3, 5), (3, 7, 64), (2, 8, 65), (1, 9, 2), (2, 63, 33), (2, 64, 130), (1, 65, 128), (3, 127, 31),
         (2, 128, 66), (1, 129, 200), (1, 1000, 7), (2, 1023, 130), (1, 2049, 64), (1, 2305, 3), (40, 5, 300), (1, 5000, 66),
         (5, 300, 257)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_training_matches_float64(R, size, dtype):
    for gate, state in ((False, False), (True, True)):
        args, gy, glast = inputs(*size, dtype, gate, state, seed=size[1])
        announce(f"gated_recurrence {size} {dtype} gate {gate} state {state}")
        want = reference(*args, 8.0, gy, glast)
        with torch.no_grad():
            y, last = train(R, *args)
        got = run(R, args, gy, glast)
        assert torch.equal(y, got["y"]) and torch.equal(last, got["last"]) and y.dtype == dtype
        for name, t in got.items():
            check(t, want[name], name)
        again = run(R, args, gy, glast)
        assert all(torch.equal(again[n], t) for n, t in got.items())  # bitwise
    no_device_errors()


def test_gates_wide_open_and_shut(R):
    """Gates at +-30: decays next to one, and down to where nothing is left."""
    args, gy, glast = inputs(2, 300, 70, torch.float32, True, True, seed=1, spread=12.0)
    args[4][:10] = torch.linspace(-60, 20, 10).cuda()
    announce("gated_recurrence extreme gates")
    want = reference(*args, 8.0, gy, glast)
    got = run(R, args, gy, glast)
    for name, t in got.items():
        assert torch.isfinite(t).all(), name
        check(t, want[name], name)
    for scale in (0.5, 30.0):
        want = reference(*args, scale, gy, glast)
        got = run(R, args, gy, glast, scale)
        for name, t in got.items():
            check(t, want[name], f"{name} at scale {scale}")


def test_parts_alone(R):
    """Gradients of one tensor at a time, and of one output at a time."""
    args, gy, glast = inputs(2, 200, 40, torch.float32, True, True, seed=2)
    full = run(R, args, gy, glast)
    announce("gated_recurrence parts alone")
    for n in NAMES:
        got = run(R, args, gy, glast, wanted=(n,))
        assert torch.equal(got[n], full[n]), n
    for a, b in ((gy, None), (None, glast)):
        want = reference(*args, 8.0, gy if a is not None else torch.zeros_like(gy), b)
        got = run(R, args, a, b)
        for n in NAMES:
            check(got[n], want[n], n)


def test_special_values_stay_in_their_channel_and_sequence(R):
    args, gy, glast = inputs(3, 400, 66, torch.float32, True, True, seed=3)
    clean = run(R, args, gy, glast)
    args[0][0, 150, 3] = float("nan")
    args[2][1, 200, 5] = float("nan")
    args[5][2, 7] = float("inf")
    announce("gated_recurrence special values")
    got = run(R, args, gy, glast)
    y = got["y"]
    assert torch.isnan(y[0, 150:, 3]).all() and torch.equal(y[0, :150, 3], clean["y"][0, :150, 3])
    assert torch.isnan(y[1, 200:, 5]).all()
    assert torch.isinf(got["last"][2, 7])  # an infinite state stays so, however many chunks decay it
    mask = torch.ones_like(y, dtype=torch.bool)
    mask[0, :, 3] = mask[1, :, 5] = mask[2, :, 7] = False
    for n in ("y", "x", "i", "r", "z"):
        assert torch.equal(got[n][mask], clean[n][mask]), n


def test_large_states_outlive_strong_decays(R):
    """1e33 under a decay of e^-80 a chunk is still 1e-2: neither factor may be lost."""
    L = 256
    x = torch.zeros(1, L, 64).cuda()
    r = torch.zeros(1, L, 64).cuda()
    k = 80.0 / 128 * 2 / 8  # l = -80 / 128 a step
    decay = torch.full((64,), float(np.log(np.expm1(k)))).cuda()
    start = torch.full((1, 64), 1e33).cuda()
    announce("gated_recurrence large states")
    want = reference(x, x, r, None, decay, start, 8.0)
    y, last = R.gated_recurrence(x, x, r, decay, None, start)
    check(y, want["y"], "y")
    check(last, want["last"], "last")
    assert last.min() > 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides_and_other_streams(R, dtype):
    """Columns of one projection (aligned and not), transposed and broadcast tensors, a side
    stream: all what dense tensors give."""
    B, L, D = 2, 150, 66
    args, gy, glast = inputs(B, L, D, dtype, True, True, seed=4)
    want, exact = run(R, args, gy, glast), reference(*args, 8.0, gy, glast)
    for off, more in ((0, 8), (2, 8), (0, 9), (1, 9), (2, 9), (3, 8)):
        wide = torch.zeros(B, L, 4 * D + more, dtype=dtype, device="cuda")
        views = [wide[..., off + k * D:off + (k + 1) * D].copy_(t) for k, t in enumerate(args[:4])]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        announce(f"gated_recurrence strided {off} {dtype}")
        with torch.cuda.stream(side):
            got = run(R, [*views, *args[4:]], gy, glast)
        torch.cuda.synchronize()
        for n, t in got.items():
            check(t, exact[n], n)
            # 16-bit rows off whole words take chunks of other lengths, and round otherwise
            assert off % 2 or more % 2 or torch.equal(t, want[n]), n
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in args[:4]]
    got = run(R, [*turned, *args[4:]], gy.transpose(0, 1).contiguous().transpose(0, 1), glast)
    assert all(torch.equal(t, want[n]) for n, t in got.items())
    one = args[1][:1, :1].expand(B, L, D)
    got = R.gated_recurrence(args[0], one, *args[2:3], args[4])
    assert torch.equal(got[0], R.gated_recurrence(args[0], one.contiguous(), args[2], args[4])[0])
    leaf = args[0].clone().requires_grad_(True)
    y, _ = R.gated_recurrence(leaf, *args[1:3], args[4])
    g1, = torch.autograd.grad(y.sum(), leaf, retain_graph=True)
    g2, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.equal(g1, g2)


def test_against_differences(R):
    """Along random directions, step 2^-7: the differences' own errors, u / step and
    step^2 of a loss of the terms' size, stay below 4e-3 of the sum of |terms|."""
    args, gy, glast = inputs(1, 40, 9, torch.float32, True, True, seed=5)
    got = run(R, args, gy, glast)

    def loss(*t):
        y, last = train(R, *t)
        return (y.double() * gy.double()).sum().item() + (last.double() * glast.double()).sum().item()

    rng = np.random.default_rng(0)
    announce("gated_recurrence against differences")
    for k, n in enumerate(NAMES):
        d = torch.tensor(rng.normal(size=args[k].shape)).float().cuda()
        h = 2.0 ** -7
        up, down = (loss(*(a + s * h * d if j == k else a for j, a in enumerate(args))) for s in (1, -1))
        terms = got[n].double() * d.double()
        assert abs((up - down) / (2 * h) - terms.sum().item()) <= 4e-3 * terms.abs().sum().item() + 4e-3, n


def test_second_derivatives(R):
    """create_graph differentiates as the separate steps do, shared tensors too."""
    args, gy, glast = inputs(2, 11, 5, torch.float32, True, True, seed=6)

    def second(f):
        leaves = [t.clone().requires_grad_(True) for t in args]
        x, i, r, z, decay, start = leaves
        y, last = f(x, i + x, r, z, decay, start)
        g = torch.autograd.grad([y, last], leaves, [gy, glast], create_graph=True)
        return torch.autograd.grad(sum((t * t).sum() for t in g), leaves)

    announce("gated_recurrence second derivatives")
    got = second(lambda *t: train(R, *t))
    want = second(lambda *t: R._separate(*t, 8.0))
    for n, p, q in zip(NAMES, got, want):
        assert (p - q).abs().max() <= 1e-4 * q.abs().max() + 1e-6, n


def test_empty_batches(R):
    announce("gated_recurrence of nothing")
    for B, L, D in ((0, 5, 4), (2, 0, 4), (2, 5, 0)):
        x = torch.zeros(B, L, D).cuda()
        state = torch.ones(B, D).cuda()
        y, last = R.gated_recurrence(x, x, x, torch.zeros(D).cuda(), None, state)
        assert y.shape == (B, L, D) and torch.equal(last, state)


# ------------------------------------------------------------------------ serving
def serve_reference(x, i, r, z, decay, pool, slots, offsets, resume, out_slots, scale=8.0):
    x, i, r, z, decay, pool = map(f64, (x, i, r, z, decay, pool))
    p = Parts(x, i, r, z, decay, scale)
    y, ty = np.zeros_like(x), np.zeros_like(x)
    after, tp = pool.copy(), np.zeros_like(pool)
    n_slots = len(pool)
    for s in range(len(offsets) - 1):
        lo, hi = offsets[s], offsets[s + 1]
        h = pool[slots[s]] if resume[s] and 0 <= slots[s] < n_slots else np.zeros(x.shape[1])
        e = np.zeros_like(h)
        for t in range(lo, hi):
            e = p.a[t] * (e + (10 * np.abs(p.l[t]) + 7) * U * np.abs(h)) + 26 * U * np.abs(p.b[t]) + M0 * np.abs(p.x[t])
            h = p.a[t] * h + p.b[t]
            y[t] = h * p.out[t]
            ty[t] = e * np.abs(p.out[t]) + 10 * U * np.abs(y[t])
        if 0 <= out_slots[s] < n_slots:
            after[out_slots[s]], tp[out_slots[s]] = h, e
    return (y, ty), (after, tp)


def serve_inputs(rows, D, slots, dtype, gate, seed):
    rng = np.random.default_rng(seed)
    packed = torch.tensor(rng.normal(size=(rows, 4 * D))).to(dtype).cuda()
    x, i, r, z = packed.chunk(4, -1)
    rate = np.exp(rng.uniform(np.log(1e-3), np.log(0.3), D))
    decay = torch.tensor(np.log(np.expm1(2 * rate / 8))).float().cuda()
    return [x, i, r, z if gate else None, decay, torch.tensor(rng.normal(size=(slots, D))).float().cuda()], rng


LENGTHS = [[1], [5], [0], [0, 0, 3], [1, 1, 1, 1], [300], [127, 1, 0, 128, 2], [1, 400, 0, 0, 77, 128, 129, 1], [5] * 60,
           [2500, 1, 700], [0] * 40 + [10] + [0] * 40]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: f"{len(v)}-{sum(v)}")
def test_prompts_match_float64(R, lengths, dtype):
    n = len(lengths)
    for D, gate, pad in ((66, True, 0), (33, False, 7), (130, True, 3)):
        rows = sum(lengths) + 2 * pad
        args, rng = serve_inputs(rows, D, 2 * n + 1, dtype, gate, seed=n + D)
        offsets = np.concatenate([[0], np.cumsum(lengths)]) + pad
        order = rng.permutation(2 * n + 1)
        slots, out_slots = order[:n].copy(), order[n:2 * n].copy()
        if n > 2:
            slots[1], out_slots[2] = -1, 2 * n + 9
        resume = rng.random(n) < 0.6
        pool = args[5].clone()
        announce(f"recurrence_prompt {n} prompts of {sum(lengths)} {dtype} D {D}")
        want_y, want_p = serve_reference(*args, slots, offsets, resume, out_slots)
        t = lambda a, d=torch.int32: torch.tensor(a).to(d).cuda()  # noqa: E731
        y = R.recurrence_prompt(*args[:3], args[4], pool, t(slots), t(offsets, torch.int64), t(resume, torch.bool),
                                output_gate=args[3], out_slots=t(out_slots))
        check(y, want_y, "y")
        check(pool, want_p, "pool")
        untouched = np.setdiff1d(np.arange(2 * n + 1), out_slots)
        assert torch.equal(pool[untouched], args[5][untouched])
        # in place, all from zeros
        pool = args[5].clone()
        want_y, want_p = serve_reference(*args, order[:n], offsets, [False] * n, order[:n])
        y = R.recurrence_prompt(*args[:3], args[4], pool, t(order[:n]), t(offsets), output_gate=args[3])
        check(y, want_y, "y")
        check(pool, want_p, "pool")
    no_device_errors()


def test_prompts_of_no_rows_and_of_no_prompts(R):
    args, _ = serve_inputs(0, 20, 3, torch.float32, False, 0)
    pool = args[5].clone()
    z = torch.zeros(3, dtype=torch.int32).cuda()
    announce("recurrence_prompt of nothing")
    y = R.recurrence_prompt(*args[:3], args[4], pool, torch.tensor([2, 0]).cuda(), z, torch.tensor([True, False]).cuda(),
                            out_slots=torch.tensor([1, 0]).cuda())
    assert y.shape == (0, 20) and torch.equal(pool[1], args[5][2]) and not pool[0].any()
    args, _ = serve_inputs(9, 20, 3, torch.float32, False, 0)
    y = R.recurrence_prompt(*args[:3], args[4], args[5], z[:0], z[:1])
    assert not y.any()


def test_a_prompts_nan_stays_its_own(R):
    lengths = [50, 90, 40, 200, 30]
    args, _ = serve_inputs(sum(lengths) + 5, 66, 5, torch.float32, True, 7)
    offsets = torch.tensor([0, *np.cumsum(lengths)]).cuda()
    slots = torch.arange(5).cuda()
    call = lambda p: R.recurrence_prompt(*args[:3], args[4], p, slots, offsets, torch.ones(5, dtype=torch.bool).cuda(),  # noqa: E731
                                         output_gate=args[3])
    clean_pool, pool = args[5].clone(), args[5].clone()
    clean = call(clean_pool)
    pool[1] = float("nan")
    args[0][200] = float("inf")
    args[2][-2:] = float("nan")  # padding
    announce("recurrence_prompt special values")
    y = call(pool)
    assert torch.isnan(y[50:140]).all() and torch.isnan(pool[1]).all() and not torch.isfinite(y[200:380]).any(1).all()
    for s in (0, 4):
        lo, hi = int(offsets[s]), int(offsets[s + 1])
        assert torch.equal(y[lo:hi], clean[lo:hi]) and torch.equal(pool[s], clean_pool[s])
    assert torch.equal(y[140:180], clean[140:180]) and not y[410:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(1, 1), (1, 2048), (3, 64), (7, 33), (65, 130), (300, 257)], ids=lambda s: "x".join(map(str, s)))
def test_steps_match_float64(R, size, dtype):
    rows, D = size
    for gate in (False, True):
        args, rng = serve_inputs(rows, D, 2 * rows + 1, dtype, gate, seed=D)
        order = rng.permutation(2 * rows + 1)
        slots, out_slots = order[:rows].copy(), order[rows:2 * rows].copy()
        if rows > 4:
            slots[1], out_slots[2] = -1, -1
            slots[3] = out_slots[3] = 2 * rows + 5  # padding
        pool = args[5].clone()
        want_y, want_p = serve_reference(*args, slots, np.arange(rows + 1), [True] * rows, out_slots)
        if rows > 4:
            want_y[0][3] = 0
        announce(f"recurrence_step {size} {dtype} gate {gate}")
        t = lambda a: torch.tensor(a).to(torch.int32).cuda()  # noqa: E731
        y = R.recurrence_step(*args[:3], args[4], pool, t(slots), output_gate=args[3], out_slots=t(out_slots))
        check(y, want_y, "y")
        check(pool, want_p, "pool")


def test_prompts_steps_and_training_agree(R):
    """The same sequence whole, as a prompt in pieces, and token by token."""
    B, L, D = 3, 300, 96
    args, *_ = inputs(B, L, D, torch.float32, True, False, seed=8)
    announce("recurrence in all its forms")
    want = reference(*args, 8.0)
    pool = torch.zeros(B, D).cuda()
    slots = torch.arange(B).cuda()
    flat = [None if t is None else t for t in args[:4]]
    cut = 257
    piece = lambda lo, hi: [t[:, lo:hi].reshape(-1, D) for t in flat]  # noqa: E731
    ends = lambda n: torch.arange(0, (B + 1) * n, n).cuda()  # noqa: E731
    x, i, r, z = piece(0, cut)
    y1 = R.recurrence_prompt(x, i, r, args[4], pool, slots, ends(cut), output_gate=z).view(B, cut, D)
    x, i, r, z = piece(cut, L - 3)
    y2 = R.recurrence_prompt(x, i, r, args[4], pool, slots, ends(L - 3 - cut), torch.ones(B, dtype=torch.bool).cuda(),
                             output_gate=z).view(B, -1, D)
    y3 = []
    for t in range(L - 3, L):
        x, i, r, z = (v[:, t] for v in flat)
        y3.append(R.recurrence_step(x, i, r, args[4], pool, slots, output_gate=z))
    check(torch.cat([y1, y2, torch.stack(y3, 1)], 1), want["y"], "y")
    check(pool, want["last"], "last")


def test_long_pools_past_32_bits(R):
    """Slots whose states start past 2^31 elements."""
    D = 1024
    n = 2 ** 21 + 3
    pool = torch.empty(n, D, device="cuda")
    pool[-2:] = torch.randn(2, D).cuda()
    args, _ = serve_inputs(6, D, 2, torch.float32, False, 9)
    small = pool[-2:].clone()
    announce("recurrence pools past 2^31 elements")
    slots = torch.tensor([n - 2, n - 1]).cuda()
    offsets = torch.tensor([0, 2, 4]).cuda()
    yes = torch.ones(2, dtype=torch.bool).cuda()
    y = R.recurrence_prompt(*(t[:4] for t in args[:3]), args[4], pool, slots, offsets, yes)
    y0 = R.recurrence_prompt(*(t[:4] for t in args[:3]), args[4], small, torch.arange(2).cuda(), offsets, yes)
    assert torch.equal(y, y0) and torch.equal(pool[-2:], small)
    y = R.recurrence_step(*(t[4:] for t in args[:3]), args[4], pool, slots)
    y0 = R.recurrence_step(*(t[4:] for t in args[:3]), args[4], small, torch.arange(2).cuda())
    assert torch.equal(y, y0) and torch.equal(pool[-2:], small)


def test_graph_capture(R):
    """Training, a prompt with offsets that change, and a step, captured after one eager call on the
    stream and replayed between eager calls, each replay against the eager result."""
    args, gy, glast = inputs(2, 500, 130, torch.float32, True, True, seed=10)
    serve, _ = serve_inputs(400, 130, 8, torch.float32, True, 11)
    offsets = torch.tensor([0, 100, 100, 390], dtype=torch.int32).cuda()
    slots, resume = torch.tensor([1, 5, 2], dtype=torch.int32).cuda(), torch.tensor([True, True, False]).cuda()
    start = serve[5].clone()

    def call():
        pool = start.clone()
        out = run(R, args, gy, glast)
        a = R.recurrence_prompt(*serve[:3], serve[4], pool, slots, offsets, resume, output_gate=serve[3])
        b = R.recurrence_step(*(t[:3] for t in serve[:3]), serve[4], pool, slots, output_gate=serve[3][:3])
        return [*out.values(), a, b, pool]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    announce("recurrence under graph capture")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    for k in range(4):
        args[0].normal_()
        serve[0].normal_()
        offsets.copy_(torch.tensor([k, 100 + k, 150, 400 - 3 * k], dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), f"replay {k}"
    no_device_errors()


def test_mixer(R):
    """The block around it: training, prompts and steps agree; its packed gradient is the separate one."""
    torch.manual_seed(0)
    m = R.RecurrentMixer(48).cuda()
    x = torch.randn(2, 70, 48).cuda()
    announce("RecurrentMixer")
    whole = m(x)
    state = R.RecurrentState.of(m, 4)
    slots = torch.tensor([3, 1]).cuda()
    with torch.no_grad():
        first = m.prompt(x[:, :69].reshape(-1, 48), state, slots, torch.tensor([0, 69, 138]).cuda()).view(2, 69, 48)
        last = m.step(x[:, 69], state, slots)
    # float32 sums of up to 96 terms in other orders: 1e-5 of the largest value
    assert (torch.cat([first, last[:, None]], 1) - whole).abs().max() <= 1e-5 * whole.abs().max()
    gy = torch.randn_like(whole)
    grads = torch.autograd.grad(m(x), list(m.parameters()), gy)
    packed = torch.nn.functional.linear(x, m.in_proj.weight)
    parts = packed.chunk(4, -1)
    y, _ = R._separate(*parts, m.decay, None, 8.0)
    want = torch.autograd.grad(torch.nn.functional.linear(y, m.out_proj.weight), list(m.parameters()), gy)
    for p, q in zip(grads, want):
        assert (p - q).abs().max() <= 1e-4 * q.abs().max()
    g = torch.autograd.grad(m(x), list(m.parameters()), gy, create_graph=True)
    h = torch.autograd.grad(sum((t * t).sum() for t in g), list(m.parameters()))
    assert all(torch.isfinite(t).all() for t in h)
    half = R.RecurrentMixer(48).cuda().bfloat16()
    half.load_state_dict(m.state_dict())
    assert (half(x.bfloat16()).float() - whole).abs().max() <= 0.1 * whole.abs().max()


def test_refusals(R):
    x, d = torch.zeros(2, 6, 8).cuda(), torch.zeros(8).cuda()
    for match, args in (("one dtype", (x.half(), x.half(), x.half(), d)), ("one dtype", (x, x.bfloat16(), x, d)),
                        ("one dtype", (x.cpu(),) * 3 + (d,)), ("all of one shape", (x, x[:1], x, d)),
                        ("all of one shape", (x[0], x[0], x[0], d)), ("decay must be", (x, x, x, d.bfloat16())),
                        ("decay must be", (x, x, x, d[:4])), ("state must be", (x, x, x, d, None, d)),
                        ("all of one shape", (x, x, x, d, x[..., :4]))):
        with pytest.raises(RuntimeError, match=match):
            R.gated_recurrence(*args)
    x, pool, s = x[0], torch.zeros(3, 8).cuda(), torch.zeros(6, dtype=torch.int32).cuda()
    for match, args in (("state is updated", (x, x, x, d, pool[:, :4], s)), ("state is updated", (x, x, x, d, pool.bfloat16(), s)),
                        ("state is updated", (x, x, x, d, torch.zeros(8, 3).cuda().t(), s)), ("slots must be", (x, x, x, d, pool, s[:5])),
                        ("int32 or int64", (x, x, x, d, pool, s.float())), ("one dtype", (x, x, x.half(), d, pool, s))):
        with pytest.raises(RuntimeError, match=match):
            R.recurrence_step(*args)
    for match, args in (("offsets must be", (x, x, x, d, pool, s, s)),
                        ("resume must be", (x, x, x, d, pool, s[:1], s[:2], torch.zeros(2, dtype=torch.bool).cuda()))):
        with pytest.raises(RuntimeError, match=match):
            R.recurrence_prompt(*args)
    for scale in (-8.0, 0.0, float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="scale must be positive"):
            R.gated_recurrence(x[None], x[None], x[None], d, scale=scale)
        with pytest.raises(RuntimeError, match="scale must be positive"):
            R.recurrence_step(x, x, x, d, pool, s, scale=scale)
        with pytest.raises(RuntimeError, match="scale must be positive"):
            R.recurrence_prompt(x, x, x, d, pool, s[:1], torch.tensor([0, 6], dtype=torch.int32).cuda(), scale=scale)
        with pytest.raises(ValueError, match="scale must be positive"):
            R.RecurrentMixer(8, scale=scale)
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="inference"):
        R.recurrence_step(leaf, x, x, d, pool, s)
    from torch.autograd import forward_ad

    announce("recurrence with tangents")
    with torch.no_grad(), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="tangent"):
            R.recurrence_step(dual, x, x, d, pool, s)
        with pytest.raises(RuntimeError, match="tangent"):
            R.gated_recurrence(dual[None], x[None], x[None], d)
