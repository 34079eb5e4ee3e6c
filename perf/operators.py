"""The operators that serve and train a language model of Mamba mixers, as measurable cases.

Four kinds of call, each through the entry point a program would use: the mixer
over ragged prompts and over single tokens with its states in a pool
(``ossm_amd.decode``), the gated projection of a feed-forward block, forward and
backward (``ossm_amd.gated``), and the penalties, biases and grammar masks on a
model's logits (``ossm_amd.logits``).
"""

import math
import random

import numpy as np
import torch

own = False

ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "sigmoid", "relu")


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # The next token of one sequence: two launches' latency, the weights and
        # one state.
        {"name": "step_one", "kind": "step", "dtype": "bf16", "S": 1, "Di": 2048, "N": 16, "R": 64, "K": 4,
         "skip": True},
        # The next token of a full serving batch: the states' traffic.
        {"name": "step_batch", "kind": "step", "dtype": "bf16", "S": 256, "Di": 2048, "N": 16, "R": 64, "K": 4,
         "skip": True},
        # One user's short prompt: the time to the first token.
        {"name": "prompt_one", "kind": "prompt", "dtype": "bf16", "T": 117, "S": 1, "Di": 2048, "N": 16, "R": 64,
         "K": 4, "skip": True, "resume": False},
        # The histories of a batch of users at the sequence-recommendation width.
        {"name": "prompt_users", "kind": "prompt", "dtype": "f32", "T": 25600, "S": 256, "Di": 128, "N": 16, "R": 4,
         "K": 4, "skip": False, "resume": False},
        # A batch of long prompts, half of them continued from an earlier piece.
        {"name": "prompt_long", "kind": "prompt", "dtype": "bf16", "T": 16384, "S": 6, "Di": 2048, "N": 16, "R": 64,
         "K": 4, "skip": True, "resume": True},
        # The feed-forward of the next token of a few sequences: the weights' traffic.
        {"name": "gated_token", "kind": "gated", "dtype": "bf16", "T": 4, "D": 2048, "F": 5632, "act": "silu",
         "bias": False, "train": False},
        # The feed-forward over a prompt, odd sizes, 32-bit weights.
        {"name": "gated_prompt_f32", "kind": "gated", "dtype": "f32", "T": 1001, "D": 1022, "F": 2730,
         "act": "gelu_tanh", "bias": True, "train": False},
        # A gated linear unit of a small recommendation model, training.
        {"name": "gated_train_f32", "kind": "gated", "dtype": "f32", "T": 25600, "D": 128, "F": 512,
         "act": "sigmoid", "bias": True, "train": True},
        # Training step of a block's gated projection: the largest case.
        {"name": "gated_train", "kind": "gated", "dtype": "bf16", "T": 8192, "D": 2048, "F": 8192, "act": "silu",
         "bias": False, "train": True},
        # One answer's next token: a row of logits, its history, a few biases.
        {"name": "logits_one", "kind": "logits", "dtype": "f32", "S": 1, "V": 50001, "H": 700, "Kb": 5,
         "mask": False},
        # A serving batch under grammars, odd vocabulary.
        {"name": "logits_grammar", "kind": "logits", "dtype": "f32", "S": 48, "V": 100003, "H": 2048, "Kb": 300,
         "mask": True},
        # A large batch, long histories, 16-bit logits.
        {"name": "logits_batch", "kind": "logits", "dtype": "bf16", "S": 256, "V": 131072, "H": 8192, "Kb": 32,
         "mask": True},
    ]


def _size(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    kind = rng.choice(("step", "prompt", "gated", "gated", "logits"))
    case = {"kind": kind, "dtype": rng.choice(("bf16", "f32"))}
    if kind in ("step", "prompt"):
        di = _size(rng, 64, 4096)
        case |= {"Di": di, "N": rng.choice((7, 8, 16, 16, 16, 32)), "R": max(1, di // 32),
                 "K": rng.choice((2, 3, 4, 4, 4, 8)), "skip": rng.random() < 0.7}
        if kind == "step":
            case["S"] = _size(rng, 1, 512)
        else:
            case["T"] = _size(rng, 1, 32768)
            case["S"] = _size(rng, 1, max(1, min(256, case["T"])))
            case["resume"] = rng.random() < 0.5
    elif kind == "gated":
        case |= {"T": _size(rng, 1, 32768), "D": _size(rng, 32, 4096), "F": _size(rng, 32, 8192),
                 "act": rng.choice(ACTIVATIONS), "bias": rng.random() < 0.5, "train": rng.random() < 0.5}
    else:
        case |= {"S": _size(rng, 1, 512), "V": _size(rng, 1000, 200000), "H": _size(rng, 1, 8192),
                 "Kb": _size(rng, 1, 512), "mask": rng.random() < 0.7}
    return case


def draw(rng):
    top = {c["kind"]: work(c) for c in listed()}  # the last of a kind is its largest
    while True:
        case = _draw_once(rng)
        if 3072 in case.values():
            continue
        w, most = work(case), top[case["kind"]]
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] / (4 if case["dtype"] == "f32" else 1):
            return case


# --------------------------------------------------------------------- inputs
class _Draws:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(self, *shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=self.g) * scale).to(dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0, dtype=torch.float32):
        return (torch.rand(*shape, device="cuda", generator=self.g) * (hi - lo) + lo).to(dtype)

    def integers(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, device="cuda", generator=self.g)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


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


def prepare(case, seed):
    make, dt, kind = _Draws(seed), _dtype(case), case["kind"]
    rng = random.Random(seed)
    state = {"case": case}
    if kind in ("step", "prompt"):
        Di, N, R, K, S = (case[k] for k in ("Di", "N", "R", "K", "S"))
        # initialised as the mixer's constructor does
        step = torch.exp(make.uniform(Di, lo=math.log(1e-3), hi=math.log(0.1)))
        state["weights"] = [
            make.uniform(Di, K, lo=-K ** -0.5, hi=K ** -0.5, dtype=dt),
            make.uniform(Di, lo=-K ** -0.5, hi=K ** -0.5, dtype=dt),
            make.uniform(R + 2 * N, Di, lo=-Di ** -0.5, hi=Di ** -0.5, dtype=dt),
            make.uniform(Di, R, lo=-R ** -0.5, hi=R ** -0.5, dtype=dt),
            step + torch.log(-torch.expm1(-step)),
            torch.log(torch.arange(1, N + 1, device="cuda", dtype=torch.float32).repeat(Di, 1)),
        ]
        state["skip"] = make.uniform(Di, lo=0.5, hi=1.5) if case["skip"] else None
        # a pool twice the batch: sequences continue from one half and, so that a
        # pass can be made again, leave their states in the other (a program that
        # forks sequences does so; others name the same slots twice)
        state["conv_state"] = make.randn(2 * S, K - 1, Di, dtype=dt)
        state["ssm_state"] = make.randn(2 * S, N, Di, scale=0.3)
        order = list(range(2 * S))
        rng.shuffle(order)
        state["slots"] = torch.tensor(order[:S], dtype=torch.int32, device="cuda")
        state["out_slots"] = torch.tensor(order[S:], dtype=torch.int32, device="cuda")
        rows = S
        if kind == "prompt":
            rows = case["T"]
            ends = np.cumsum([0] + _lengths(case, rng))
            state["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
            state["resume"] = None
            if case["resume"]:
                state["resume"] = torch.tensor([i % 2 == 0 for i in range(S)], device="cuda")
        state["xz"] = make.randn(rows, 2 * Di, dtype=dt)
    elif kind == "gated":
        T, D, F = case["T"], case["D"], case["F"]
        s = 2 * D ** -0.5
        state["x"] = make.randn(T, D, dtype=dt)
        state["weights"] = [make.uniform(F, D, lo=-s, hi=s, dtype=dt), make.uniform(F, D, lo=-s, hi=s, dtype=dt)]
        state["biases"] = [make.uniform(F, lo=-s, hi=s, dtype=dt) if case["bias"] else None for _ in range(2)]
        if case["train"]:
            state["go"] = make.randn(T, F, dtype=dt)
            for t in (state["x"], *state["weights"], *state["biases"]):
                if t is not None:
                    t.requires_grad_(True)
    else:
        S, V, H, Kb = (case[k] for k in ("S", "V", "H", "Kb"))
        state["logits"] = make.randn(S, V, scale=3.0, dtype=dt)
        # few distinct words make up most of a text
        ids = (make.uniform(S, H) ** 6 * V).long().clamp_(max=V - 1)
        state["history"] = ids.to(torch.int32)
        state["lengths"] = make.integers(H // 2, H + 1, S).to(torch.int32)
        state["prompt_lengths"] = make.integers(0, H // 2 + 1, S).to(torch.int32)
        state["repetition"] = make.uniform(S, lo=1.0, hi=1.5)
        state["presence"] = make.uniform(S, lo=0.0, hi=1.0)
        state["frequency"] = make.uniform(S, lo=0.0, hi=0.5)
        # distinct ids: one to each of Kb stretches of the vocabulary
        Kb = min(Kb, V)
        edges = torch.arange(Kb, device="cuda") * (V // Kb)
        state["bias_ids"] = (edges + make.integers(0, V // Kb, S, Kb)).to(torch.int32)
        state["bias_values"] = make.randn(S, Kb, scale=4.0)
        # a grammar allows one word in eight
        state["allowed"] = None
        if case["mask"]:
            words = [make.integers(-2 ** 31, 2 ** 31, S, (V + 31) // 32) for _ in range(3)]
            state["allowed"] = (words[0] & words[1] & words[2]).to(torch.int32)
    return state


# ------------------------------------------------------------- the plain forms
def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _act(name, a):
    """The activation and its derivative."""
    if name == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    if name == "sigmoid":
        s = torch.sigmoid(a)
        return s, s * (1 - s)
    if name == "relu":
        return torch.clamp(a, min=0), (a > 0).to(a.dtype)
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(a * 0.5 ** 0.5))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) * (2 * math.pi) ** -0.5
    c, k = (2 / math.pi) ** 0.5, 0.044715
    t = torch.tanh(c * (a + k * a ** 3))
    return 0.5 * a * (1 + t), 0.5 * (1 + t) + 0.5 * a * (1 - t * t) * c * (1 + 3 * k * a * a)


def _mixer_parts(st, u, z):
    """Decays [rows, N, Di], inputs and read-outs of the state update."""
    cw, cb, xw, dw, db, a_log = st["weights"]
    N, R = st["case"]["N"], st["case"]["R"]
    proj = u @ xw.float().t()
    dt = _softplus(proj[:, :R] @ dw.float().t() + db)
    decay = torch.exp(dt.unsqueeze(1) * -torch.exp(a_log).t())
    push = proj[:, R:R + N].unsqueeze(2) * (dt * u).unsqueeze(1)
    return decay, push, proj[:, R + N:]


def _mixer_out(st, h, read, u, z):
    y = (h * read.unsqueeze(2)).sum(1)
    if st["skip"] is not None:
        y = y + st["skip"] * u
    return (y * z * torch.sigmoid(z)).to(st["xz"].dtype)


def _plain_step(st):
    Di, K = st["case"]["Di"], st["case"]["K"]
    slots, outs = st["slots"].long(), st["out_slots"].long()
    cw, cb = st["weights"][0].float(), st["weights"][1].float()
    window = torch.cat([st["conv_state"][slots], st["xz"][:, None, :Di]], 1)
    pre = (window.float() * cw.t()).sum(1) + cb
    u, z = pre * torch.sigmoid(pre), st["xz"][:, Di:].float()
    decay, push, read = _mixer_parts(st, u, z)
    h = decay * st["ssm_state"][slots] + push
    st["conv_state"][outs] = window[:, 1:]
    st["ssm_state"][outs] = h
    return [_mixer_out(st, h, read, u, z), st["conv_state"], st["ssm_state"]]


def _plain_prompt(st):
    Di, K, T, S = (st["case"][k] for k in ("Di", "K", "T", "S"))
    slots, outs, offsets = st["slots"].long(), st["out_slots"].long(), st["offsets"].long()
    cw, cb = st["weights"][0].float(), st["weights"][1].float()
    token = torch.arange(T, device=offsets.device)
    seq = torch.searchsorted(offsets, token, right=True) - 1
    resume = torch.zeros(S, dtype=torch.bool, device=offsets.device) if st["resume"] is None else st["resume"]
    # every sequence after the K - 1 inputs before it
    ext = torch.zeros(T + S * (K - 1), Di, dtype=st["xz"].dtype, device=offsets.device)
    at = token + (seq + 1) * (K - 1)
    ext[at] = st["xz"][:, :Di]
    back = torch.arange(K - 1, device=offsets.device)
    first = offsets[:-1] + torch.arange(S, device=offsets.device) * (K - 1)
    ext[first[:, None] + back] = st["conv_state"][slots] * resume[:, None, None]
    taps = at[:, None] - (K - 1) + torch.arange(K, device=offsets.device)
    pre = (ext[taps].float() * cw.t()).sum(1) + cb
    u, z = pre * torch.sigmoid(pre), st["xz"][:, Di:].float()
    decay, h, read = _mixer_parts(st, u, z)
    # h_t = decay_t h_{t-1} + push_t by doubling; a first token takes its
    # sequence's initial state and nothing from the token before it
    h0 = st["ssm_state"][slots] * resume[:, None, None]
    start = offsets[:-1][offsets[1:] > offsets[:-1]]
    h[start] += decay[start] * h0[offsets[1:] > offsets[:-1]]
    decay[start] = 0
    span = 1
    while span < T:
        h[span:] += decay[span:] * h[:-span]
        decay[span:] = decay[span:] * decay[:-span]
        span *= 2
    last = (offsets[1:] - 1).clamp(min=0)
    empty = (offsets[1:] == offsets[:-1])[:, None, None]
    st["conv_state"][outs] = ext[first[:, None] + (offsets[1:] - offsets[:-1])[:, None] + back]
    st["ssm_state"][outs] = torch.where(empty, h0, h[last])
    return [_mixer_out(st, h, read, u, z), st["conv_state"], st["ssm_state"]]


def _plain_gated(st):
    case, dt = st["case"], st["x"].dtype
    x, (wg, wu) = st["x"].detach().float(), (w.detach().float() for w in st["weights"])
    a, b = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        a, b = a + st["biases"][0].detach().float(), b + st["biases"][1].detach().float()
    f, df = _act(case["act"], a)
    y = f * b
    if not case["train"]:
        return y.to(dt)
    go = st["go"].float()
    da, db = go * b * df, go * f
    grads = [da @ wg + db @ wu, da.t() @ x, db.t() @ x]
    if case["bias"]:
        grads += [da.sum(0), db.sum(0)]
    return [y.to(dt)] + [g.to(dt) for g in grads]


def _plain_logits(st):
    S, V = st["case"]["S"], st["case"]["V"]
    logits = st["logits"].float()
    at = torch.arange(st["history"].size(1), device=logits.device)
    ids = st["history"].long()
    seen = torch.zeros_like(logits).scatter_add_(1, ids, (at < st["lengths"][:, None]).float())
    said = (at < st["lengths"][:, None]) & (at >= st["prompt_lengths"][:, None])
    said = torch.zeros_like(logits).scatter_add_(1, ids, said.float())
    rep = st["repetition"][:, None]
    out = torch.where(seen > 0, torch.where(logits > 0, logits / rep, logits * rep), logits)
    out = out - st["frequency"][:, None] * said - st["presence"][:, None] * (said > 0).float()
    out = out.scatter_add_(1, st["bias_ids"].long(), st["bias_values"])
    if st["allowed"] is not None:
        v = torch.arange(V, device=logits.device)
        bit = (st["allowed"][:, v // 32] >> (v % 32).to(torch.int32)) & 1
        out = torch.where(bit == 1, out, float("-inf"))
    return out.to(st["logits"].dtype)


# ------------------------------------------------------------------- the call
def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return {"step": _plain_step, "prompt": _plain_prompt, "gated": _plain_gated,
                "logits": _plain_logits}[kind](state)
    if kind == "step":
        from ossm_amd.decode import mixer_step
        y = mixer_step(state["xz"], *state["weights"], state["conv_state"], state["ssm_state"], state["slots"],
                       skip=state["skip"], out_slots=state["out_slots"])
        return [y, state["conv_state"], state["ssm_state"]]
    if kind == "prompt":
        from ossm_amd.decode import mixer_prompt
        y = mixer_prompt(state["xz"], *state["weights"], state["conv_state"], state["ssm_state"], state["slots"],
                         state["offsets"], state["resume"], skip=state["skip"], out_slots=state["out_slots"])
        return [y, state["conv_state"], state["ssm_state"]]
    if kind == "gated":
        from ossm_amd.gated import gated_linear
        with torch.set_grad_enabled(case["train"]):
            y = gated_linear(state["x"], *state["weights"], *state["biases"], activation=case["act"])
            if not case["train"]:
                return y
            ins = [state["x"], *state["weights"], *(t for t in state["biases"] if t is not None)]
            return [y.detach(), *torch.autograd.grad(y, ins, state["go"])]
    from ossm_amd.logits import control_logits
    return control_logits(state["logits"], state["history"], state["lengths"], state["prompt_lengths"],
                          repetition=state["repetition"], presence=state["presence"],
                          frequency=state["frequency"], bias_ids=state["bias_ids"],
                          bias_values=state["bias_values"], allowed=state["allowed"])


# ----------------------------------------------------------------------- work
def work(case):
    """Every input read once and every output written once, no intermediate; the
    operations of the products and, per state and step, the decay's exponential and
    product, the input's product and sum, the read-out's (7)."""
    e, kind = (2 if case["dtype"] == "bf16" else 4), case["kind"]
    if kind in ("step", "prompt"):
        Di, N, R, K, S = (case[k] for k in ("Di", "N", "R", "K", "S"))
        rows = S if kind == "step" else case["T"]
        read = S if kind == "step" else (S + 1) // 2 if case["resume"] else 0
        weights = e * Di * (K + 1 + 2 * R + 2 * N) + 4 * Di * (N + 2)
        states = (S + read) * Di * (4 * N + e * (K - 1))
        return {"bytes": 3 * e * rows * Di + weights + states,
                "flops": rows * Di * (2 * K + 2 * (2 * R + 2 * N) + 7 * N + 16)}
    if kind == "gated":
        T, D, F = case["T"], case["D"], case["F"]
        once = T * D + 2 * F * D + (2 * F if case["bias"] else 0)
        # the backward takes the two input gradients' and the two weights' products
        return {"bytes": e * (once * (2 if case["train"] else 1) + T * F * (2 if case["train"] else 1)),
                "flops": 4 * T * D * F * (3 if case["train"] else 1) + 12 * T * F}
    S, V, H, Kb = (case[k] for k in ("S", "V", "H", "Kb"))
    return {"bytes": S * (2 * e * V + 4 * H + 8 * Kb + (V // 8 if case["mask"] else 0)), "flops": S * (6 * V + H)}


# ----------------------------------------------------- the same in 64 bits
def _exact_mixer(st, rows_of, conv0, h0):
    """Sequence by sequence, token by token; rows_of[i] are sequence i's rows of xz.  The
    products are taken over all rows at once (they do not depend on the order)."""
    case = st["case"]
    Di, N, R, K = (case[k] for k in ("Di", "N", "R", "K"))
    cw, cb, xw, dw, db, a_log = (w.double() for w in st["weights"])
    xz = st["xz"].double()
    u = torch.empty(xz.size(0), Di, dtype=torch.float64, device=xz.device)
    tails = []
    for i, (lo, hi) in enumerate(rows_of):
        full = torch.cat([conv0[i].double(), xz[lo:hi, :Di]])
        pre = cb.expand(hi - lo, Di).clone()
        for k in range(K):
            pre += cw[:, k] * full[k:k + hi - lo]
        u[lo:hi] = pre / (1 + torch.exp(-pre))
        tails.append(full[full.size(0) - (K - 1):])
    proj = u @ xw.t().contiguous()
    dt = torch.nn.functional.softplus(proj[:, :R] @ dw.t().contiguous() + db, threshold=40.0)
    A = -torch.exp(a_log).t()
    h = h0.double().clone()  # [sequences, N, Di]
    y = torch.empty_like(u)
    order = sorted(range(len(rows_of)), key=lambda i: rows_of[i][0] - rows_of[i][1])
    lo = torch.tensor([rows_of[i][0] for i in order], device=xz.device)
    lengths = [rows_of[i][1] - rows_of[i][0] for i in order]
    h = h[torch.tensor(order, device=xz.device)]
    live = len(order)
    for t in range(max(lengths)):
        while live and lengths[live - 1] <= t:
            live -= 1
        r = lo[:live] + t
        hn = torch.exp(A * dt[r].unsqueeze(1)) * h[:live] + (dt[r] * u[r]).unsqueeze(1) * proj[r, R:R + N, None]
        h[:live] = hn
        y[r] = torch.bmm(proj[r, None, R + N:], hn).squeeze(1)
    back = torch.empty_like(h)
    back[torch.tensor(order, device=xz.device)] = h
    if st["skip"] is not None:
        y = y + st["skip"].double() * u
    z = xz[:, Di:]
    conv, ssm = st["conv_state"].double(), st["ssm_state"].double()
    for i, slot in enumerate(st["out_slots"].tolist()):
        conv[slot], ssm[slot] = tails[i], back[i]
    return [y * z / (1 + torch.exp(-z)), conv, ssm]


def _exact_gated(st):
    case = st["case"]
    x, wg, wu = (t.detach().double().requires_grad_(case["train"]) for t in (st["x"], *st["weights"]))
    bias = [t.detach().double().requires_grad_(case["train"]) for t in st["biases"] if t is not None]
    nf = torch.nn.functional
    a, b = nf.linear(x, wg, *bias[:1]), nf.linear(x, wu, *bias[1:])
    f = {"silu": nf.silu, "gelu": nf.gelu, "gelu_tanh": lambda t: nf.gelu(t, approximate="tanh"),
         "sigmoid": torch.sigmoid, "relu": nf.relu}[case["act"]](a)
    y = f * b
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, [x, wg, wu, *bias], st["go"].double())]


def _exact_logits(st):
    V = st["case"]["V"]
    get = lambda k: st[k].cpu().numpy()  # noqa: E731
    out = st["logits"].double().cpu().numpy()
    rows = zip(out, get("history"), get("lengths"), get("prompt_lengths"), get("repetition"), get("presence"),
               get("frequency"), get("bias_ids"), get("bias_values"))
    for i, (row, hist, n, first, rep, pres, freq, ids, values) in enumerate(rows):
        words = np.unique(hist[:n])
        row[words] = np.where(row[words] > 0, row[words] / np.float64(rep), row[words] * np.float64(rep))
        count = np.bincount(hist[first:n], minlength=V).astype(np.float64) if n > first else np.zeros(V)
        row -= np.float64(freq) * count + np.float64(pres) * (count > 0)
        row[ids] += values.astype(np.float64)
        if st["allowed"] is not None:
            bits = np.unpackbits(st["allowed"][i].cpu().numpy().view(np.uint8), bitorder="little")[:V]
            row[bits == 0] = -np.inf
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "logits":
        return _exact_logits(st)
    if case["kind"] == "gated":
        return _exact_gated(st)
    with torch.no_grad():
        slots = st["slots"].long()
        conv0, h0 = st["conv_state"][slots], st["ssm_state"][slots]
        if case["kind"] == "step":
            return _exact_mixer(st, [(i, i + 1) for i in range(case["S"])], conv0, h0)
        keep = torch.zeros(case["S"], device=h0.device) if st["resume"] is None else st["resume"].float()
        ends = st["offsets"].tolist()
        return _exact_mixer(st, list(zip(ends, ends[1:])), conv0 * keep[:, None, None].to(conv0.dtype),
                            h0 * keep[:, None, None])
