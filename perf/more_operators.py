"""Further operators of a recurrent language model, as measurable cases.

Three kinds of call, each through the entry point a program would use: layer norm,
alone or of a residual sum, forward and backward (``ossm_amd.norm``); the gated linear
recurrence over training batches, ragged prompts and single tokens
(``ossm_amd.recurrence``); and the choice of the next token by temperature, top-k,
top-p and min-p from given random numbers (``ossm_amd.sampling``).
"""

import math
import random

import numpy as np
import torch

own = False

SCALE = 8.0  # the recurrence's decay at a wide open gate is exp(-SCALE softplus(decay))


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # The norm before a block of the next token of a few sequences: latency.
        {"name": "norm_token", "kind": "norm", "dtype": "bf16", "wdtype": "bf16", "T": 4, "D": 2048, "residual": True,
         "train": False},
        # A prompt's norm in 32 bits, odd sizes.
        {"name": "norm_prompt_f32", "kind": "norm", "dtype": "f32", "wdtype": "f32", "T": 1001, "D": 1023,
         "residual": False, "train": False},
        # A small recommendation model's norm, training: many short rows.
        {"name": "norm_train_f32", "kind": "norm", "dtype": "f32", "wdtype": "f32", "T": 25600, "D": 128,
         "residual": True, "train": True},
        # Training step of a large model's norm after its residual sum, weights kept in 32 bits.
        {"name": "norm_train", "kind": "norm", "dtype": "bf16", "wdtype": "f32", "T": 32768, "D": 2048,
         "residual": True, "train": True},
        # The next token of a serving batch: states in a pool, one launch's latency.
        {"name": "recur_step", "kind": "step", "dtype": "bf16", "S": 32, "D": 2048, "gate": True},
        # The histories of a batch of users at the sequence-recommendation width.
        {"name": "recur_prompt_users", "kind": "prompt", "dtype": "f32", "T": 25600, "S": 256, "D": 128, "gate": False,
         "resume": False},
        # A batch of long prompts, half of them continued from an earlier piece.
        {"name": "recur_prompt_long", "kind": "prompt", "dtype": "bf16", "T": 16384, "S": 6, "D": 2048, "gate": True,
         "resume": True},
        # Training step of a small model in 32 bits, odd sizes, from given states.
        {"name": "recur_train_f32", "kind": "recur", "dtype": "f32", "B": 16, "L": 1001, "D": 257, "gate": False,
         "state": True},
        # Training step of a large model's recurrence with its output gate: the largest case.
        {"name": "recur_train", "kind": "recur", "dtype": "bf16", "B": 4, "L": 8192, "D": 2048, "gate": True,
         "state": False},
        # One answer's next token.
        {"name": "sample_one", "kind": "sample", "dtype": "f32", "S": 1, "V": 50001, "k": True, "p": True, "m": False,
         "mask": False, "rows": False},
        # A serving batch under grammars, each request with settings of its own, odd vocabulary.
        {"name": "sample_mixed", "kind": "sample", "dtype": "f32", "S": 48, "V": 100003, "k": True, "p": True, "m": True,
         "mask": True, "rows": True},
        # A large batch, 16-bit logits: many ties.
        {"name": "sample_batch", "kind": "sample", "dtype": "bf16", "S": 256, "V": 131072, "k": False, "p": True,
         "m": True, "mask": False, "rows": True},
    ]


def _size(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    kind = rng.choice(("norm", "norm", "step", "prompt", "recur", "sample", "sample"))
    case = {"kind": kind, "dtype": rng.choice(("bf16", "f32"))}
    if kind == "norm":
        case |= {"wdtype": rng.choice(("f32", case["dtype"])), "T": _size(rng, 1, 65536), "D": _size(rng, 1, 16384),
                 "residual": rng.random() < 0.6, "train": rng.random() < 0.6}
    elif kind == "step":
        case |= {"S": _size(rng, 1, 1024), "D": _size(rng, 16, 8192), "gate": rng.random() < 0.6}
    elif kind == "prompt":
        case |= {"T": _size(rng, 1, 65536), "D": _size(rng, 16, 8192), "gate": rng.random() < 0.6,
                 "resume": rng.random() < 0.5}
        case["S"] = _size(rng, 1, max(1, min(512, case["T"])))
    elif kind == "recur":
        case |= {"B": _size(rng, 1, 64), "L": _size(rng, 1, 16384), "D": _size(rng, 16, 4096),
                 "gate": rng.random() < 0.6, "state": rng.random() < 0.5}
    else:
        case |= {"S": _size(rng, 1, 512), "V": _size(rng, 100, 262144), "k": rng.random() < 0.5,
                 "p": rng.random() < 0.6, "m": rng.random() < 0.4, "mask": rng.random() < 0.4,
                 "rows": rng.random() < 0.7}
    return case


def draw(rng):
    top = {c["kind"]: work(c) for c in listed()}  # the last of a kind is its largest
    top["step"] = {k: 32 * v for k, v in top["step"].items()}
    while True:
        case = _draw_once(rng)
        w, most = work(case), top[case["kind"]]
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return case


# --------------------------------------------------------------------- inputs
class _Draws:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(self, *shape, scale=1.0, shift=0.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=self.g) * scale + shift).to(dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0, dtype=torch.float32):
        return (torch.rand(*shape, device="cuda", generator=self.g) * (hi - lo) + lo).to(dtype)

    def integers(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, device="cuda", generator=self.g)


def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _lengths(case, rng):
    """S lengths that add up to T, very uneven, one of them empty where there are several."""
    T, S = case["T"], case["S"]
    weights = [rng.expovariate(1.0) + 0.05 for _ in range(S)]
    if S >= 4:
        weights[rng.randrange(S)] = 0.0
    total = sum(weights)
    lengths = [int(T * w / total) for w in weights]
    lengths[weights.index(max(weights))] += T - sum(lengths)
    return lengths


def _decay(make, D):
    """Decays as a model starts from: at a gate half open a channel remembers 5 to 2000 steps."""
    rate = torch.exp(make.uniform(D, lo=math.log(5e-4), hi=math.log(0.2)))
    return torch.log(torch.expm1(2 * rate / SCALE))


def prepare(case, seed):
    make, dt, kind = _Draws(seed), _type(case["dtype"]), case["kind"]
    rng = random.Random(seed)
    st = {"case": case}
    if kind == "norm":
        T, D, wdt = case["T"], case["D"], _type(case["wdtype"])
        st["x"] = make.randn(T, D, dtype=dt)
        # a residual stream is wider than what a block adds, and off centre
        st["residual"] = make.randn(T, D, scale=3.0, shift=0.5, dtype=dt) if case["residual"] else None
        st["weight"], st["bias"] = make.randn(D, scale=0.2, shift=1.0, dtype=wdt), make.randn(D, scale=0.2, dtype=wdt)
        if case["train"]:
            st["gy"] = make.randn(T, D, dtype=dt)
            st["gs"] = make.randn(T, D, dtype=dt) if case["residual"] else None
            for t in (st["x"], st["residual"], st["weight"], st["bias"]):
                if t is not None:
                    t.requires_grad_(True)
    elif kind in ("step", "prompt", "recur"):
        D = case["D"]
        shape = {"step": lambda: (case["S"],), "prompt": lambda: (case["T"],),
                 "recur": lambda: (case["B"], case["L"])}[kind]()
        # one projection's columns, as a mixer makes them: input, its gate, the decay's gate, the output's
        parts = make.randn(*shape, (4 if case["gate"] else 3) * D, dtype=dt).split(D, -1)
        st["decay"] = _decay(make, D)
        if kind == "recur":
            st["x"], st["i"], st["r"] = (t.contiguous().requires_grad_(True) for t in parts[:3])
            st["z"] = parts[3].contiguous().requires_grad_(True) if case["gate"] else None
            st["decay"].requires_grad_(True)
            st["h0"] = make.randn(case["B"], D).requires_grad_(True) if case["state"] else None
            st["gy"] = make.randn(*shape, D, dtype=dt)
            st["glast"] = make.randn(case["B"], D)
            return st
        st["x"], st["i"], st["r"] = parts[:3]
        st["z"] = parts[3] if case["gate"] else None
        # a pool twice the batch: sequences continue from one half and, so that a
        # pass can be made again, leave their states in the other
        S = case["S"]
        order = list(range(2 * S))
        rng.shuffle(order)
        st["pool"] = make.randn(2 * S, D)
        st["slots"] = torch.tensor(order[:S], dtype=torch.int32, device="cuda")
        st["out_slots"] = torch.tensor(order[S:], dtype=torch.int32, device="cuda")
        if kind == "prompt":
            ends = np.cumsum([0] + _lengths(case, rng))
            st["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
            st["resume"] = None
            if case["resume"]:
                st["resume"] = torch.tensor([i % 2 == 0 for i in range(S)], device="cuda")
    else:
        S, V = case["S"], case["V"]
        st["logits"] = make.randn(S, V, scale=3.0, dtype=dt)
        if case["mask"]:  # a grammar allows one word in eight
            forbidden = make.integers(0, 8, S, V) != 0
            forbidden[:, 0] = False
            st["logits"].masked_fill_(forbidden, float("-inf"))
        st["u"] = make.uniform(S)
        if case["rows"]:
            # every request has settings of its own; some are greedy, some leave a filter off
            off = lambda t, v: torch.where(make.uniform(S) < 0.1, torch.full_like(t, v), t)  # noqa: E731
            st["temperature"] = off(make.uniform(S, lo=0.5, hi=1.2), 0.0)
            st["top_k"] = off(torch.exp(make.uniform(S, lo=0.0, hi=math.log(min(V, 2000)))).to(torch.int32), 0) \
                if case["k"] else None
            st["top_p"] = off(make.uniform(S, lo=0.3, hi=0.99), 1.0) if case["p"] else None
            st["min_p"] = off(torch.exp(make.uniform(S, lo=math.log(1e-3), hi=math.log(0.3))), 0.0) \
                if case["m"] else None
        else:
            # one request's numbers (a setting is a 32-bit number, given alone or in a tensor)
            number = lambda *of: float(np.float32(rng.choice(of)))  # noqa: E731
            st["temperature"] = number(0.6, 0.7, 0.8, 1.0)
            st["top_k"] = min(V, rng.choice((20, 50, 200))) if case["k"] else None
            st["top_p"] = number(0.8, 0.9, 0.95) if case["p"] else None
            st["min_p"] = number(0.01, 0.05, 0.1) if case["m"] else None
    return st


# ------------------------------------------------------------- the plain forms
def _plain_norm(st):
    case, dt, wdt = st["case"], st["x"].dtype, st["weight"].dtype
    s = st["x"].detach().float()
    if case["residual"]:
        s = (s + st["residual"].detach().float()).to(dt).float()
    w, b = st["weight"].detach().float(), st["bias"].detach().float()
    c = s - s.mean(1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5)
    xhat = c * rstd
    out = [(xhat * w + b).to(dt)] + ([s.to(dt)] if case["residual"] else [])
    if not case["train"]:
        return out
    gy = st["gy"].float()
    g = gy * w
    ds = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if case["residual"]:
        ds = (ds + st["gs"].float()).to(dt)
        out += [ds, ds]
    else:
        out.append(ds.to(dt))
    return out + [(gy * xhat).sum(0).to(wdt), gy.sum(0).to(wdt)]


def _doubling(a, h, t):
    """h_t += a_t h_{t-1} along axis t, in place, by doubling the span."""
    n, span = a.size(t), 1
    while span < n:
        late, early = a.narrow(t, span, n - span), a.narrow(t, 0, n - span)
        h.narrow(t, span, n - span).add_(late * h.narrow(t, 0, n - span))
        late.copy_(late * early)
        span *= 2


def _recur_parts(st):
    """log-decay, decay, the input's factor and its gate, in 32 bits."""
    lam = st["decay"].detach().float()
    soft = torch.clamp(lam, min=0) + torch.log1p(torch.exp(-lam.abs()))
    la = -SCALE * soft * torch.sigmoid(st["r"].detach().float())
    return la, torch.exp(la), torch.sqrt(-torch.expm1(2 * la)), torch.sigmoid(st["i"].detach().float())


def _out_gate(st, h):
    if st["z"] is None:
        return h
    z = st["z"].detach().float()
    return h * z * torch.sigmoid(z)


def _plain_step(st):
    _, a, m, gi = _recur_parts(st)
    h = a * st["pool"][st["slots"].long()] + m * gi * st["x"].float()
    st["pool"][st["out_slots"].long()] = h
    return [_out_gate(st, h).to(st["x"].dtype), st["pool"]]


def _plain_prompt(st):
    _, a, m, gi = _recur_parts(st)
    S, offsets = st["case"]["S"], st["offsets"].long()
    h = m * gi * st["x"].float()
    h0 = st["pool"][st["slots"].long()]
    h0 = torch.zeros_like(h0) if st["resume"] is None else h0 * st["resume"][:, None]
    # a first token takes its sequence's state and nothing from the token before it
    some = offsets[1:] > offsets[:-1]
    start = offsets[:-1][some]
    h[start] += a[start] * h0[some]
    a[start] = 0
    _doubling(a, h, 0)
    st["pool"][st["out_slots"].long()] = torch.where(some[:, None], h[(offsets[1:] - 1).clamp(min=0)], h0)
    return [_out_gate(st, h).to(st["x"].dtype), st["pool"]]


def _plain_recur(st):
    case, dt = st["case"], st["x"].dtype
    la, a, m, gi = _recur_parts(st)
    x = st["x"].detach().float()
    h0 = torch.zeros(case["B"], case["D"], device=x.device) if st["h0"] is None else st["h0"].detach()
    h = m * gi * x
    h[:, 0] += a[:, 0] * h0
    _doubling(a.clone(), h, 1)
    out = [_out_gate(st, h).to(dt), h[:, -1].clone()]
    go, gz = st["gy"].float(), None
    if case["gate"]:
        z = st["z"].detach().float()
        s = torch.sigmoid(z)
        gz = (go * h * s * (1 + z * (1 - s))).to(dt)
        go = go * z * s
    # G_t = go_t + a_{t+1} G_{t+1}, in reverse
    G = go.flip(1)
    G[:, 0] += st["glast"]
    back = torch.zeros_like(a)
    back[:, 1:] = a[:, 1:].flip(1)
    _doubling(back, G, 1)
    G = G.flip(1)
    del back
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    q = G * (before * a * la + gi * x * torch.where(m > 0, a * a * -la / m, torch.zeros_like(m)))
    lam = st["decay"].detach().float()
    soft = torch.clamp(lam, min=0) + torch.log1p(torch.exp(-lam.abs()))
    out += [(G * m * gi).to(dt), (G * m * x * gi * (1 - gi)).to(dt),
            (q * (1 - torch.sigmoid(st["r"].detach().float()))).to(dt),
            torch.sigmoid(lam) / soft * q.sum((0, 1))]
    if case["gate"]:
        out.append(gz)
    if st["h0"] is not None:
        out.append(a[:, 0] * G[:, 0])
    return out


def _plain_sample(st):
    # 64 bits: a token next to a border of the chosen interval must not move
    logits, u = st["logits"].double(), st["u"].double()[:, None]
    S, V = logits.shape
    col = lambda v: v.double()[:, None] if isinstance(v, torch.Tensor) else v  # noqa: E731
    t = col(st["temperature"])
    t = torch.full((S, 1), t, dtype=torch.float64, device=logits.device) if isinstance(t, float) else t
    greedy = t <= 0
    top = logits.max(1, keepdim=True).values
    w = torch.exp((logits - top) / torch.where(greedy, 1.0, t))
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(V, device=logits.device)
    keep = ws > 0
    if st["top_k"] is not None:
        k = st["top_k"][:, None] if isinstance(st["top_k"], torch.Tensor) else st["top_k"]
        keep &= (rank < k) | (torch.as_tensor(k) <= 0).to(rank.device)
    if st["top_p"] is not None:
        p = col(st["top_p"])
        some = ws * keep
        before = some.cumsum(1) - some
        keep &= (before < p * some.sum(1, keepdim=True)) | (torch.as_tensor(p) >= 1).to(rank.device)
    if st["min_p"] is not None:
        keep &= ws >= col(st["min_p"])
    keep[:, 0] = True
    w = w * torch.zeros_like(keep).scatter_(1, order, keep)
    cum = w.cumsum(1)
    token = (cum > u * cum[:, -1:]).to(torch.int8).argmax(1)
    return torch.where(greedy[:, 0], order[:, 0], token)


# ------------------------------------------------------------------- the call
def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return {"norm": _plain_norm, "step": _plain_step, "prompt": _plain_prompt, "recur": _plain_recur,
                "sample": _plain_sample}[kind](state)
    if kind == "norm":
        from ossm_amd.norm import add_layer_norm, layer_norm
        with torch.set_grad_enabled(case["train"]):
            if not case["residual"]:
                out = [layer_norm(state["x"], state["weight"], state["bias"])]
                ins, grads = [state["x"]], [state["gy"]] if case["train"] else []
            else:
                out = list(add_layer_norm(state["x"], state["residual"], state["weight"], state["bias"]))
                ins = [state["x"], state["residual"]]
                grads = [state["gy"], state["gs"]] if case["train"] else []
            if not case["train"]:
                return out
            return [t.detach() for t in out] + \
                list(torch.autograd.grad(out, [*ins, state["weight"], state["bias"]], grads))
    if kind == "step":
        from ossm_amd.recurrence import recurrence_step
        y = recurrence_step(state["x"], state["i"], state["r"], state["decay"], state["pool"], state["slots"],
                            output_gate=state["z"], scale=SCALE, out_slots=state["out_slots"])
        return [y, state["pool"]]
    if kind == "prompt":
        from ossm_amd.recurrence import recurrence_prompt
        y = recurrence_prompt(state["x"], state["i"], state["r"], state["decay"], state["pool"], state["slots"],
                              state["offsets"], state["resume"], output_gate=state["z"], scale=SCALE,
                              out_slots=state["out_slots"])
        return [y, state["pool"]]
    if kind == "recur":
        from ossm_amd.recurrence import gated_recurrence
        y, last = gated_recurrence(state["x"], state["i"], state["r"], state["decay"], state["z"], state["h0"],
                                   scale=SCALE)
        ins = [t for t in (state["x"], state["i"], state["r"], state["decay"], state["z"], state["h0"])
               if t is not None]
        return [y.detach(), last.detach(), *torch.autograd.grad([y, last], ins, [state["gy"], state["glast"]])]
    from ossm_amd.sampling import sample_logits
    return sample_logits(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                         top_p=state["top_p"], min_p=state["min_p"])


# ----------------------------------------------------------------------- work
def work(case):
    """Every input read once and every output written once, no intermediate; an exponential,
    a root and a quotient count as one operation each."""
    e, kind = (2 if case["dtype"] == "bf16" else 4), case["kind"]
    if kind == "norm":
        T, D, we = case["T"], case["D"], 2 if case["wdtype"] == "bf16" else 4
        forward = 4 if case["residual"] else 2
        backward = (3 if case["residual"] else 2) if case["train"] else 0  # gy, gs and the gradient
        return {"bytes": e * T * D * (forward + backward) + we * D * (4 if case["train"] else 2),
                "flops": T * D * (9 + (14 if case["train"] else 0))}
    if kind in ("step", "prompt"):
        D, rows = case["D"], case["S"] if kind == "step" else case["T"]
        read = case["S"] if kind == "step" else (case["S"] + 1) // 2 if case["resume"] else 0
        n = 5 if case["gate"] else 4
        return {"bytes": e * rows * D * n + 4 * D * (case["S"] + read + 1), "flops": rows * D * (20 + 5 * (n - 4))}
    if kind == "recur":
        n, D = case["B"] * case["L"] * case["D"], case["D"]
        tensors = 5 + 4 if case["gate"] else 4 + 4  # forward, then the gradients of each input and the output's
        tensors += 1 if case["gate"] else 0
        return {"bytes": e * n * tensors + 8 * D + 4 * case["B"] * D * (4 if case["state"] else 2),
                "flops": n * (20 + 30 + (12 if case["gate"] else 0))}
    S, V = case["S"], case["V"]
    return {"bytes": S * (e * V + 32), "flops": 8 * S * V}


# ----------------------------------------------------- the same in 64 bits
def _exact_norm(st):
    case, dt = st["case"], st["x"].dtype
    nf = torch.nn.functional
    s = st["x"].detach().double()
    if case["residual"]:
        s = (s + st["residual"].detach().double()).to(dt).double()
    s.requires_grad_(case["train"])
    w, b = (t.detach().double().requires_grad_(case["train"]) for t in (st["weight"], st["bias"]))
    y = nf.layer_norm(s, (case["D"],), w, b, 1e-5)
    out = [y.detach()] + ([s.detach()] if case["residual"] else [])
    if not case["train"]:
        return out
    ds, dw, db = torch.autograd.grad(y, [s, w, b], st["gy"].double())
    if case["residual"]:
        ds = ds + st["gs"].double()
    return out + [ds] * (2 if case["residual"] else 1) + [dw, db]


def _exact_parts(lam, i, r, x):
    """decays and inputs of the recurrence from its definition."""
    a = torch.exp(-SCALE * torch.nn.functional.softplus(lam, threshold=40.0) * torch.sigmoid(r))
    # (1 - a)(1 + a) loses nothing that 64 bits hold at the decays of these inputs
    return a, torch.sqrt((1 - a) * (1 + a)) * torch.sigmoid(i) * x


def _exact_served(st, rows_of, h0):
    case = st["case"]
    x, i, r, lam = (st[k].double() for k in ("x", "i", "r", "decay"))
    a, b = _exact_parts(lam, i, r, x)
    order = sorted(range(len(rows_of)), key=lambda s: rows_of[s][0] - rows_of[s][1])
    at = torch.tensor(order, device=x.device)
    lo = torch.tensor([rows_of[s][0] for s in order], device=x.device)
    lengths = [rows_of[s][1] - rows_of[s][0] for s in order]
    h, hs, live = h0.double()[at], torch.zeros_like(b), len(order)
    for t in range(max(lengths)):
        while live and lengths[live - 1] <= t:
            live -= 1
        rows = lo[:live] + t
        h[:live] = a[rows] * h[:live] + b[rows]
        hs[rows] = h[:live]
    pool = st["pool"].double()
    pool[st["out_slots"].long()[at]] = h
    y = hs * torch.nn.functional.silu(st["z"].double()) if case["gate"] else hs
    return [y, pool]


def _exact_recur(st):
    case = st["case"]
    ins = {k: None if st[k] is None else st[k].detach().double().requires_grad_(True)
           for k in ("x", "i", "r", "decay", "z", "h0")}
    a, b = _exact_parts(ins["decay"], ins["i"], ins["r"], ins["x"])
    h = ins["h0"] if ins["h0"] is not None else torch.zeros_like(a[:, 0])
    hs = []
    for at, bt in zip(a.unbind(1), b.unbind(1)):
        h = at * h + bt
        hs.append(h)
    y = torch.stack(hs, 1)
    if case["gate"]:
        y = y * torch.nn.functional.silu(ins["z"])
    wanted = [t for t in ins.values() if t is not None]
    grads = torch.autograd.grad([y, h], wanted, [st["gy"].double(), st["glast"].double()])
    return [y.detach(), h.detach(), *grads]


def _exact_sample(st):
    logits, u = st["logits"].double().cpu().numpy(), st["u"].double().cpu().numpy()
    S, V = logits.shape
    get = lambda v, i: v[i].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    given = {k: st[k].cpu() if isinstance(st[k], torch.Tensor) else st[k]
             for k in ("temperature", "top_k", "top_p", "min_p")}
    out = np.empty(S, np.int64)
    for i, row in enumerate(logits):
        t, k, p, m = (get(v, i) for v in given.values())
        if t <= 0:
            out[i] = row.argmax()
            continue
        ids = np.argsort(-row, kind="stable")
        ids = ids[row[ids] > -np.inf]
        if k is not None and k > 0:
            ids = ids[:k]
        w = np.exp(((row[ids] - row[ids[0]]) / t).astype(np.longdouble))
        if p is not None and p < 1:
            cum = np.cumsum(w)
            n = 1 + int(np.searchsorted(cum[:-1], p * cum[-1], side="left"))
            ids, w = ids[:n], w[:n]
        if m is not None:
            n = max(1, int((w >= m).sum()))
            ids, w = ids[:n], w[:n]
        back = np.argsort(ids)
        cum = np.cumsum(w[back])
        out[i] = ids[back][np.searchsorted(cum, u[i] * cum[-1], side="right")]
    return out


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "norm":
        return _exact_norm(st)
    if kind == "sample":
        return _exact_sample(st)
    if kind == "recur":
        return _exact_recur(st)
    with torch.no_grad():
        h0 = st["pool"][st["slots"].long()]
        if kind == "step":
            return _exact_served(st, [(s, s + 1) for s in range(case["S"])], h0)
        keep = torch.zeros(case["S"], device=h0.device) if st["resume"] is None else st["resume"].float()
        ends = st["offsets"].tolist()
        return _exact_served(st, list(zip(ends, ends[1:])), h0 * keep[:, None])
