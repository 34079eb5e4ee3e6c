"""GPU tests of the served Mamba mixer (ossm_amd.decode): ragged prompts and single
tokens with their states in a pool, against a token-by-token float64 computation.

Tolerances, derived before the first run: everything is computed in float32, sums
of up to Di = 300 products (x_proj) and of up to N = 40 (the read-out), states that
remember about 1 / (1 - decay) tokens.  Their roundings stay below 64 of float32's
half ulps of the largest value of the same kind: 64 * 2^-24 = 4e-6, and 2e-5 of the
tensor's largest value bounds that with the hardware exponentials' error (2^-22 of
each).  A bfloat16 output adds its own rounding, 2^-8 of the value (half ulp 2^-9,
with room for a neighbour's tie)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.gpu_util import announce, need_gpu, no_device_errors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def D():
    need_gpu()
    from ossm_amd import decode

    return decode


class Case:
    """Weights, a pool and packed inputs, on the GPU."""

    def __init__(self, Di, N, R, K, lengths, dtype=torch.float32, seed=0, slots=None, skip=True, bias=True, pad=0,
                 n_slots=None):
        rng = np.random.default_rng(seed)
        f = lambda *s, scale=1.0: torch.tensor(rng.normal(size=s) * scale, dtype=torch.float32)  # noqa: E731
        self.Di, self.N, self.R, self.K, self.lengths = Di, N, R, K, list(lengths)
        S = len(lengths)
        self.S, self.rows = S, sum(lengths) + pad
        w = [f(Di, 1, K, scale=0.5), f(Di, scale=0.2) if bias else None, f(R + 2 * N, Di, scale=Di ** -0.5),
             f(Di, R, scale=R ** -0.5), torch.tensor(rng.uniform(-5, -1, Di), dtype=torch.float32),
             torch.log(torch.arange(1, N + 1, dtype=torch.float32)).repeat(Di, 1) + f(Di, N, scale=0.1)]
        cast = lambda t: None if t is None else t.to(dtype).cuda()  # noqa: E731
        self.w = [cast(t) for t in w[:4]] + [t.cuda() for t in w[4:]]
        self.skip = f(Di).cuda() if skip else None
        n_slots = n_slots or 2 * S + 1
        self.conv, self.ssm = f(n_slots, K - 1, Di).to(dtype).cuda(), f(n_slots, N, Di).cuda()
        order = rng.permutation(n_slots)
        self.slots = torch.tensor(order[:S] if slots is None else slots, dtype=torch.int32).cuda()
        self.offsets = torch.tensor(np.cumsum([0] + self.lengths), dtype=torch.int32).cuda()
        self.xz = f(self.rows, 2 * Di).to(dtype).cuda()
        self.resume = torch.tensor(rng.random(S) < 0.5).cuda()

    def args(self, conv=None, ssm=None):
        return (*self.w, self.conv if conv is None else conv, self.ssm if ssm is None else ssm, self.slots)


def reference(c, resume, out_slots=None):
    """float64 on the CPU, one sequence and one token at a time: (y, conv pool, ssm pool)."""
    d = lambda t: None if t is None else t.detach().double().cpu().numpy()  # noqa: E731
    cw, cb, xp, dp, db, al = (d(t) for t in c.w)
    cw = cw.reshape(c.Di, c.K)
    A = -np.exp(al).T
    conv, ssm, xz = d(c.conv), d(c.ssm), d(c.xz)
    conv0, ssm0 = conv.copy(), ssm.copy()
    slots = c.slots.tolist()
    outs = slots if out_slots is None else out_slots.tolist()
    y = np.zeros((c.rows, c.Di))
    skip = np.zeros(c.Di) if c.skip is None else d(c.skip)
    t = 0
    for s, n in enumerate(c.lengths):
        keep = 0 <= slots[s] < len(ssm) and bool(resume[s])
        win = conv0[slots[s]].copy() if keep else np.zeros((c.K - 1, c.Di))
        h = ssm0[slots[s]].copy() if keep else np.zeros((c.N, c.Di))
        for _ in range(n):
            full = np.concatenate([win, xz[t:t + 1, :c.Di]])
            pre = np.sum(full * cw.T, 0) + (0 if cb is None else cb)
            u = pre / (1 + np.exp(-pre))
            p = xp @ u
            dt = np.logaddexp(0, dp @ p[:c.R] + db)
            h = np.exp(A * dt) * h + np.outer(p[c.R:c.R + c.N], dt * u)
            z = xz[t, c.Di:]
            y[t] = (p[c.R + c.N:] @ h + skip * u) * z / (1 + np.exp(-z))
            win = full[1:]
            t += 1
        if 0 <= outs[s] < len(ssm):
            conv[outs[s]], ssm[outs[s]] = win, h
    return y, conv, ssm


def check(got, want, dtype=torch.float32, what=""):
    g = got.detach().double().cpu().numpy()
    assert g.shape == want.shape
    tol = 2e-5 * max(np.abs(want).max(initial=0.0), 1e-3) + (2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0)
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())}/{bad.size} off, worst {np.abs(g - want).max():.3e}"


def run_prompt(D, c, resume=None, **kw):
    return D.mixer_prompt(c.xz, *c.args(), c.offsets, resume, skip=c.skip, **kw)


SIZES = [  # Di, N, R, K
    (1, 1, 1, 1), (5, 3, 2, 2), (64, 16, 4, 4), (130, 7, 9, 3), (128, 16, 8, 4), (300, 16, 10, 4), (96, 40, 6, 4),
    (200, 33, 5, 8), (67, 32, 64, 5)]
LENGTHS = [[1], [2, 1, 3], [0], [0, 5, 0, 0, 1, 0], [517], [15, 16, 17, 1, 0, 64, 33], [200, 0, 1, 130]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_prompt_matches_float64(D, size, dtype):
    """Every length pattern, from zeros and half of them resumed; states in place."""
    for i, lengths in enumerate(LENGTHS):
        for resumed in (False, True):
            c = Case(*size, lengths, dtype, seed=i, skip=i % 2 == 0, bias=i % 3 != 0)
            announce(f"mixer_prompt {size} {lengths} {dtype} resumed={resumed}")
            want = reference(c, c.resume.tolist() if resumed else [False] * c.S)
            y = run_prompt(D, c, c.resume if resumed else None)
            check(y, want[0], dtype, "y")
            check(c.conv, want[1], torch.float32, "conv state")  # copies: no rounding
            check(c.ssm, want[2], torch.float32, "ssm state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 31, 32, 77])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_step_matches_float64(D, size, rows, dtype):
    c = Case(*size, [1] * rows, dtype, seed=rows)
    announce(f"mixer_step {size} rows={rows} {dtype}")
    want = reference(c, [True] * rows)
    y = D.mixer_step(c.xz, *c.args(), skip=c.skip)
    check(y, want[0], dtype, "y")
    check(c.conv, want[1], torch.float32, "conv state")
    check(c.ssm, want[2], torch.float32, "ssm state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size, lengths", [
    ((600, 16, 10, 4), [700, 0, 1, 1300, 15]),  # over a hundred chunks: dt by its own kernel, chunks in groups
    ((1030, 40, 33, 5), [513, 1, 700, 2]),  # two passes over the states, odd ranks
    ((128, 16, 8, 4), [9000, 3, 17, 160])], ids=["600", "1030", "128"])
def test_large_prompts(D, size, lengths, dtype):
    for resumed in (False, True):
        c = Case(*size, lengths, dtype, seed=20, pad=9)
        announce(f"mixer_prompt {size} {lengths} {dtype} resumed={resumed}")
        want = reference(c, c.resume.tolist() if resumed else [False] * c.S)
        y = run_prompt(D, c, c.resume if resumed else None)
        check(y, want[0], dtype, "y")
        check(c.conv, want[1], torch.float32, "conv state")
        check(c.ssm, want[2], torch.float32, "ssm state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(600, 16, 38, 4), (1030, 40, 33, 5)], ids=["600", "1030"])
def test_large_steps(D, size, dtype):
    c = Case(*size, [1] * 301, dtype, seed=21)
    announce(f"mixer_step {size} rows=301 {dtype}")
    want = reference(c, [True] * 301)
    y = D.mixer_step(c.xz, *c.args(), skip=c.skip)
    check(y, want[0], dtype, "y")
    check(c.conv, want[1], torch.float32, "conv state")
    check(c.ssm, want[2], torch.float32, "ssm state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("channels", [103000, 263000])  # weights shared by the projection, and by the scan
@pytest.mark.parametrize("size", [s for s in SIZES if s[0] >= 64], ids=lambda s: "x".join(map(str, s)))
def test_steps_of_many_sequences(D, size, channels, dtype):
    rows = channels // size[0] + 2
    c = Case(*size, [1] * rows, dtype, seed=23, skip=channels < 200000, bias=channels > 200000)
    announce(f"mixer_step {size} rows={rows} {dtype}")
    want = reference(c, [True] * rows)
    y = D.mixer_step(c.xz, *c.args(), skip=c.skip)
    check(y, want[0], dtype, "y")
    check(c.conv, want[1], torch.float32, "conv state")
    check(c.ssm, want[2], torch.float32, "ssm state")


@pytest.mark.parametrize("Di", [128, 130])
def test_slots_and_values_among_many_sequences(D, Di):
    """Padding, rows from zeros, rows that keep nothing; NaN in one row leaves the others' bits."""
    rows = 2100
    c = Case(Di, 16, 8, 4, [1] * rows, seed=24)
    c.slots[1], c.slots[3] = -1, 10 ** 6
    used = set(c.slots.tolist())
    outs = torch.tensor([s for s in range(c.ssm.size(0)) if s not in used][:rows], dtype=torch.int32).cuda()
    outs[2], outs[3] = -1, -1
    announce(f"mixer_step among {rows} sequences, d_inner {Di}")
    want = reference(c, [True] * rows, outs)
    want[0][3] = 0  # padding
    conv, ssm = c.conv.clone(), c.ssm.clone()
    y = D.mixer_step(c.xz, *c.args(), skip=c.skip, out_slots=outs)
    for got, w in zip((y, c.conv, c.ssm), want):
        check(got, w)
    bad = c.xz.clone()
    bad[40] = float("nan")
    z = D.mixer_step(bad, *c.args(conv, ssm), skip=c.skip, out_slots=outs)
    keep = [i for i in range(rows) if i != 40]
    assert torch.equal(y[keep], z[keep]) and torch.isnan(z[40]).all()
    others = [s for s in range(ssm.size(0)) if s != int(outs[40])]
    assert torch.equal(c.ssm[others], ssm[others]) and torch.isnan(ssm[int(outs[40])]).all()


def test_values_of_one_large_prompt_stay_in_it(D):
    lengths = [700, 800, 900]
    a, b = Case(600, 16, 10, 4, lengths, seed=22), Case(600, 16, 10, 4, lengths, seed=22)
    b.xz[900] = float("nan")  # in the second prompt
    announce("mixer_prompt of three large prompts, NaN in one")
    ya, yb = run_prompt(D, a), run_prompt(D, b)
    assert torch.equal(ya[:900], yb[:900]) and torch.equal(ya[1500:], yb[1500:])
    assert torch.isnan(yb[900:1500]).all()
    others = [s for s in range(a.ssm.size(0)) if s != int(a.slots[1])]
    assert torch.equal(a.ssm[others], b.ssm[others]) and torch.isnan(b.ssm[int(a.slots[1])]).all()


@pytest.mark.parametrize("rows", [4, 40])
def test_slots_outside_the_pool_and_forks(D, rows):
    """-1 starts from zeros or keeps nothing; a row with neither is padding; other out
    slots leave the sources as they were."""
    c = Case(64, 16, 4, 4, [1] * rows, seed=5)
    c.slots[1] = -1
    c.slots[3] = 10 ** 6
    outs = torch.tensor([s for s in range(c.ssm.size(0)) if s not in c.slots.tolist()][:rows], dtype=torch.int32).cuda()
    outs[2], outs[3] = -1, -1
    announce("mixer_step slots outside the pool")
    want = reference(c, [True] * rows, outs)
    want[0][3] = 0  # padding
    y = D.mixer_step(c.xz, *c.args(), skip=c.skip, out_slots=outs.long())
    for got, w in zip((y, c.conv, c.ssm), want):
        check(got, w)
    c = Case(64, 16, 4, 4, [3, 0, 40, 7, 0, 90], seed=6)
    c.slots[0] = -1
    outs = torch.tensor([s for s in range(c.ssm.size(0)) if s not in c.slots.tolist()][:c.S], dtype=torch.int32).cuda()
    outs[2] = 99
    announce("mixer_prompt slots outside the pool")
    want = reference(c, c.resume.tolist(), outs)
    y = run_prompt(D, c, c.resume, out_slots=outs)
    for got, w in zip((y, c.conv, c.ssm), want):
        check(got, w)


def test_a_prompt_in_pieces_then_tokens(D):
    """A prompt cut anywhere, continued, then single tokens, gives what the whole does."""
    Di, N, R, K, n = 128, 16, 8, 4, 300
    whole = Case(Di, N, R, K, [n], seed=7)
    want = reference(whole, [False])
    for cuts in ([1, 2, 297], [150, 150], [299, 1], [0, 300]):
        c = Case(Di, N, R, K, [n], seed=7)
        announce(f"mixer_prompt in pieces {cuts}")
        at, out = 0, []
        for i, m in enumerate(cuts):
            off = torch.tensor([0, m], dtype=torch.int32).cuda()
            out.append(D.mixer_prompt(c.xz[at:at + m], *c.args(), off, torch.tensor([i > 0]).cuda(), skip=c.skip))
            at += m
        for got, w in zip((torch.cat(out), c.conv, c.ssm), want):
            check(got, w)
    c = Case(Di, N, R, K, [n], seed=7)
    announce("mixer_prompt then mixer_step")
    off = torch.tensor([0, n - 9], dtype=torch.int32).cuda()
    out = [D.mixer_prompt(c.xz[:n - 9], *c.args(), off, skip=c.skip)]
    out += [D.mixer_step(c.xz[t:t + 1], *c.args(), skip=c.skip) for t in range(n - 9, n)]
    for got, w in zip((torch.cat(out), c.conv, c.ssm), want):
        check(got, w)


def test_prompt_matches_the_training_mixer(D):
    """What MambaMixer.forward gives for a batch of equal lengths, padding rows zero."""
    from ossm_amd.mamba import MambaMixer, MixerCoreFn

    torch.manual_seed(0)
    m = MambaMixer(32, d_state=16, d_conv=4, expand=2).cuda()
    B, L = 3, 50
    xz = torch.randn(B, L, 2 * m.d_inner, device="cuda")
    announce("mixer_prompt against MixerCoreFn")
    with torch.no_grad():
        w = (m.conv1d.weight, m.conv1d.bias, m.x_proj.weight, m.dt_proj.weight, m.dt_proj.bias, m.A_log)
        want = MixerCoreFn.apply(xz, *w).reshape(B * L, -1)
        st = D.MixerState.of(m, B)
        packed = torch.cat([xz.reshape(B * L, -1), torch.full((5, 2 * m.d_inner), float("nan"), device="cuda")])
        y = D.mixer_prompt(packed, *w, st.conv, st.ssm, torch.arange(B).cuda(), torch.arange(0, B * L + 1, L).cuda())
    check(y[:B * L], want.double().cpu().numpy())
    assert torch.all(y[B * L:] == 0)
    no_device_errors()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_values_of_one_sequence_stay_in_it(D, value):
    lengths = [40, 1, 0, 30, 50]
    a, b = Case(64, 16, 4, 4, lengths, seed=8), Case(64, 16, 4, 4, lengths, seed=8)
    b.xz[45] = value  # in the fourth prompt
    announce(f"mixer_prompt with {value}")
    ya, yb = run_prompt(D, a), run_prompt(D, b)
    assert torch.equal(ya[:45], yb[:45]) and torch.equal(ya[71:], yb[71:])
    others = [s for s in range(a.ssm.size(0)) if s != int(a.slots[3])]
    assert torch.equal(a.ssm[others], b.ssm[others]) and torch.equal(a.conv[others], b.conv[others])
    assert not torch.isfinite(b.ssm[int(a.slots[3])]).all()


def test_strides_streams_and_repeats(D):
    """A strided xz, another stream, and bitwise equal results of repeated calls."""
    c = Case(130, 16, 9, 4, [70, 0, 33, 140], torch.bfloat16, seed=9)
    wide = torch.full((c.rows, 2 * c.Di + 11), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 3:3 + 2 * c.Di] = c.xz
    first = None
    for i in range(3):
        conv, ssm = c.conv.clone(), c.ssm.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        announce(f"mixer_prompt strided, side stream, repeat {i}")
        with torch.cuda.stream(side if i else torch.cuda.current_stream()):
            xz = wide[:, 3:3 + 2 * c.Di] if i else c.xz
            y = D.mixer_prompt(xz, *c.args(conv, ssm), c.offsets, c.resume, skip=c.skip)
            step = D.mixer_step(xz[:4], *c.args(conv, ssm), skip=c.skip)
        torch.cuda.synchronize()
        got = [y, step, conv, ssm]
        first = first or got
        assert all(torch.equal(p, q) for p, q in zip(first, got))


def test_graph_capture(D):
    """Steps captured and replayed, with eager work between the replays."""
    c = Case(128, 16, 8, 4, [1] * 40, torch.bfloat16, seed=10)
    e = Case(128, 16, 8, 4, [1] * 40, torch.bfloat16, seed=10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    announce("mixer_step under graph capture")
    conv, ssm = c.conv.clone(), c.ssm.clone()
    with torch.cuda.stream(side):
        D.mixer_step(c.xz, *c.args(conv, ssm), skip=c.skip)  # the workspace grows before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = D.mixer_step(c.xz, *c.args(), skip=c.skip)
    for i in range(4):
        x = torch.randn_like(c.xz)
        c.xz.copy_(x)
        e.xz.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = D.mixer_step(e.xz, *e.args(), skip=e.skip)
        assert torch.equal(y, want) and torch.equal(c.ssm, e.ssm) and torch.equal(c.conv, e.conv), f"replay {i}"


def test_pool_past_32_bits(D):
    """A slot whose state lies past 2^31 elements, and past 2^32 bytes, of its pool."""
    Di, N, K, n = 4096, 16, 4, 33000
    c = Case(Di, N, 8, K, [1, 1, 1], torch.bfloat16, seed=11)
    big_conv = torch.empty(n, K - 1, Di, dtype=torch.bfloat16, device="cuda")
    big_ssm = torch.empty(n, N, Di, device="cuda")
    assert (n - 1) * N * Di > 2 ** 31
    at = torch.tensor([n - 1, 3, n - 2], dtype=torch.int32).cuda()
    big_conv[at.long()], big_ssm[at.long()] = c.conv[c.slots.long()], c.ssm[c.slots.long()]
    announce("mixer_step in a pool past 2^31 elements")
    y = D.mixer_step(c.xz, *c.w, big_conv, big_ssm, at, skip=c.skip)
    want = D.mixer_step(c.xz, *c.args(), skip=c.skip)
    assert torch.equal(y, want)
    assert torch.equal(big_ssm[at.long()], c.ssm[c.slots.long()])
    assert torch.equal(big_conv[at.long()], c.conv[c.slots.long()])


def test_no_rows_and_no_sequences(D):
    c = Case(64, 16, 4, 4, [0, 0], seed=12)
    none = torch.zeros(0, dtype=torch.int32).cuda()
    announce("mixer calls without rows")
    before = c.ssm.clone()
    assert D.mixer_step(c.xz, *c.w, c.conv, c.ssm, none).shape == (0, 64)
    assert D.mixer_prompt(c.xz, *c.w, c.conv, c.ssm, none, torch.zeros(1, dtype=torch.int32).cuda()).shape == (0, 64)
    assert torch.equal(before, c.ssm)
    run_prompt(D, c)  # two empty prompts: their slots are cleared
    assert torch.all(c.ssm[c.slots.long()] == 0) and torch.all(c.conv[c.slots.long()] == 0)


def test_refusals(D):
    c = Case(64, 16, 4, 4, [2, 3], seed=13)
    a = list(c.args())

    def refuse(match, i, v, xz=c.xz, offsets=c.offsets, **kw):
        b = list(a)
        if i is not None:
            b[i] = v
        with pytest.raises(RuntimeError, match=match):
            D.mixer_prompt(xz, *b, offsets, skip=kw.pop("skip", c.skip), **kw)

    refuse("float32 or bfloat16 GPU", None, None, xz=c.xz.half())
    refuse("inconsistent shapes", None, None, xz=c.xz[:, :-1])
    refuse("inconsistent shapes", 2, c.w[2][:-1])
    refuse("inconsistent shapes", 6, c.conv[:, :-1])
    refuse("must be torch.float32", 3, c.w[3].bfloat16())
    refuse("float32", 7, c.ssm.double())
    refuse("contiguous", 7, torch.empty(5, 64, 16, device="cuda").transpose(1, 2))
    refuse("slots must be int32", 8, c.slots.float())
    refuse("offsets must be", None, None, offsets=c.offsets[:-1])
    refuse("resume must be", None, None, resume=c.resume.float())
    refuse("must be torch.float32", 4, c.w[4].cpu())
    with pytest.raises(RuntimeError, match="inference"):
        D.mixer_step(c.xz[:2].clone().requires_grad_(True), *a)
    with pytest.raises(RuntimeError, match="conv widths"):
        e = Case(64, 16, 4, 9, [2])
        run_prompt(D, e)
    with pytest.raises(RuntimeError, match="slots must be a 1-D tensor of 5"):
        D.mixer_step(c.xz, *a)


def test_forward_mode_is_refused(D):
    """A tangent raises, under no_grad too, whichever argument carries it."""
    from torch.autograd import forward_ad

    c = Case(64, 16, 4, 4, [1, 1], seed=14)
    announce("mixer calls with tangents")
    given = [c.xz, *c.w, c.conv, c.ssm]
    with forward_ad.dual_level(), torch.no_grad():
        run_prompt(D, c)
        for i, t in enumerate((*given, c.skip)):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else u for j, u in enumerate((*given, c.skip))]
            with pytest.raises(RuntimeError, match="tangents"):
                D.mixer_step(*dual[:-1], c.slots, skip=dual[-1])
            with pytest.raises(RuntimeError, match="tangents"):
                D.mixer_prompt(*dual[:-1], c.slots, c.offsets, skip=dual[-1])


def _mixer():
    from ossm_amd.mamba import MambaMixer

    torch.manual_seed(3)
    return MambaMixer(24, d_state=8, d_conv=4, expand=2).cuda()


def _served(D, m, x):
    """What a mixer answers to x [1, L, d_model] as a prompt of all but the last two and two steps."""
    st, slot = D.MixerState.of(m, 1), torch.zeros(1, dtype=torch.int32).cuda()
    L = x.size(1)
    head = D.prompt(m, x[0, :-2], st, slot, torch.tensor([0, L - 2], dtype=torch.int32).cuda())
    return torch.cat([head, *(D.step(m, x[0, t:t + 1], st, slot) for t in (L - 2, L - 1))])


@torch.random.fork_rng()  # later tests draw what they drew
def test_a_skip_that_the_mixer_does_not_train_is_not_served(D):
    """MambaMixer.forward has no D skip, whatever its ``D`` holds."""
    m = _mixer()
    m.D = torch.nn.Parameter(torch.randn(48).cuda())
    x = torch.randn(1, 30, 24).cuda()
    announce("decode of a mixer with D set")
    with torch.no_grad():
        check(_served(D, m, x), m(x)[0].double().cpu().numpy(), what="mixer with D")


@torch.random.fork_rng()  # later tests draw what they drew
@pytest.mark.parametrize("how", ["bias", "hook", "replaced"])
def test_an_x_proj_that_is_more_than_its_weight_is_refused(D, how):
    m = _mixer()
    if how == "bias":
        m.x_proj = torch.nn.Linear(48, m.x_proj.out_features).cuda()
    elif how == "hook":
        m.x_proj.register_forward_hook(lambda mod, args, out: 2 * out)
    else:
        m.x_proj = torch.nn.Sequential(m.x_proj, torch.nn.Identity())
    x = torch.randn(1, 30, 24).cuda()
    announce(f"decode of a mixer, x_proj {how}")
    with pytest.raises(RuntimeError, match="x_proj"):
        _served(D, m, x)
    st, slot = D.MixerState.of(m, 1), torch.zeros(1, dtype=torch.int32).cuda()
    with pytest.raises(RuntimeError, match="x_proj"):
        D.step(m, x[0, :1], st, slot)


@torch.random.fork_rng()  # later tests draw what they drew
def test_a_computed_x_proj_weight_is_served(D):
    """A parametrized weight is the module's weight: what trains is what answers."""
    m = _mixer()
    torch.nn.utils.parametrizations.weight_norm(m.x_proj)
    x = torch.randn(1, 30, 24).cuda()
    announce("decode of a mixer, x_proj parametrized")
    with torch.no_grad():
        m.x_proj.parametrizations.weight.original0.mul_(1.5)
        check(_served(D, m, x), m(x)[0].double().cpu().numpy(), what="mixer with a parametrized x_proj")


@pytest.mark.parametrize("rows", [64, 400])
def test_states_past_the_range_of_a_chunks_decay(D, rows):
    """exp(A sum dt) of a chunk of tokens leaves float32's range where its product with the
    state does not (1e33 under e^-96), and an infinite state stays infinite.  The exponent of
    138 binary digits is rounded in 16 steps, 138 * 16 * 2^-24 * ln 2 = 9e-5 of the state."""
    c = Case(64, 3, 1, 1, [rows], seed=15, skip=False, bias=False)
    cw, _, xp, dp, db, al = c.w
    for t, v in ((cw, 1), (xp, 0), (dp, 1), (db, -8), (al, 0)):
        t.fill_(v)
    # p = (u_0, for dt; u_1 = 0 for B: nothing is added to the state; u_2 = 1.3 for C)
    xp[0, 0], xp[1:4, 1], xp[4:, 2] = 1, 1, 1
    c.xz[:, :3] = torch.tensor([-30.0, 0.0, 1.6]).cuda()
    c.xz[17:31, 0] = 6.857 + 8  # 14 tokens of one chunk, whatever its ends: dt = 6.857
    for value in (1e33, float("inf"), -float("inf")):
        c.ssm.fill_(value)
        announce(f"mixer_prompt of {rows} rows from states of {value}")
        with np.errstate(invalid="ignore"):
            want = reference(c, [True])
        y = run_prompt(D, c, torch.ones(1, dtype=torch.bool).cuda()).double().cpu().numpy()
        np.testing.assert_allclose(y, want[0], rtol=5e-4)
        np.testing.assert_allclose(c.ssm[c.slots.long()].double().cpu().numpy(), want[2][c.slots.tolist()], rtol=5e-4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_step_in_tiles_of_an_odd_number_of_sums(D, dtype):
    """Rows in tiles whose projections' sums are no multiple of four: what lies behind them in
    the workspace is stored in vectors."""
    Di, N, R, rows = 2184, 7, 69, 299  # 18 blocks of channels x 299 x 83 sums, 2 over a multiple of 4
    assert -(-Di // 128) * rows * (R + 2 * N) % 4 == 2
    c = Case(Di, N, R, 4, [1] * rows, dtype, seed=16)
    announce(f"mixer_step tiles, odd sums {dtype}")
    want = reference(c, [True] * rows)
    y = D.mixer_step(c.xz, *c.args(), skip=c.skip)
    check(y, want[0], dtype, "y")
    check(c.conv, want[1], torch.float32, "conv state")
    check(c.ssm, want[2], torch.float32, "ssm state")
