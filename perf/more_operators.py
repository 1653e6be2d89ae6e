"""Performance cases of the operators of a selective state space layer, beside the TTT inner loops and the gated linear
recurrence: a layer that remembers through a state per channel has its users run

    conv    causal depthwise convolution of 2 to 4 taps with bias and SiLU on [B, T, C], the last inputs carried from call to call
    scan    h_t = exp(d_t A) h_{t-1} + d_t B_t x_t,  y_t = C_t h_t + D x_t, times SiLU(z_t): N states per channel, decays that the
            token chooses (d_t = softplus(dt_t + bias)); whole sequences and steps of a few tokens
    norm    group norm with channels last: of every token's channel groups, or of a whole sequence's, times SiLU(gate) or with an
            activation of its own

forward, or forward + backward.  `run` computes a case in elementary torch operations, or through the framework's entry points
where `own` is set.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BASE = {"dtype": "bf16", "grad": False}
MORE = {
    "conv": {"K": 4, "act": "silu", "bias": True, "carry": False, "starts": False, "columns": False},
    "scan": {"N": 16, "G": 1, "gate": True, "skip": True, "carry": False, "starts": False},
    "norm": {"act": "silu", "gate": True, "over": "token", "affine": True},
}


def _case(name, op, B, T, C, **more):
    c = dict(BASE, **MORE[op], op=op, B=B, T=T, C=C)
    c.update(more)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # a generated token of a small batch: the call a serving loop repeats for each layer and token
        _case("conv-token-b8", "conv", 8, 1, 1536, carry=True),
        # a few prompts of odd length, columns of the input projection, no gradients: time to the first token
        _case("conv-prompt-odd", "conv", 3, 1201, 1536, columns=True),
        # training at the tokens of the headline workload, twice its width
        _case("conv-train-b32", "conv", 32, 2048, 1536, grad=True),
        # a generated token of a small batch and of a large one: resident states of 16 values per channel
        _case("scan-token-b8", "scan", 8, 1, 1536, carry=True),
        _case("scan-token-b128", "scan", 128, 1, 1536, carry=True),
        # one very long prompt: fewer channels than the card has lanes
        _case("scan-prompt-long", "scan", 1, 32768, 1536),
        # training
        _case("scan-train-b16", "scan", 16, 2048, 1536, grad=True),
        # float32 (parity and debugging runs) on documents packed one behind the other, state and gradient carried, two groups
        # of B and C, no gate, an odd length
        _case("scan-train-f32-docs", "scan", 2, 515, 200, N=8, G=2, dtype="f32", grad=True, gate=False, carry=True, starts=True),
        # a generated token of a small batch: heads of 64 features normed and gated
        _case("norm-token-b8", "norm", 8, 1, 1536, groups=24),
        # training, every token's heads
        _case("norm-train-b32", "norm", 32, 2048, 1536, groups=24, grad=True),
        # training of a layer that sees its whole sequence at once: statistics over all of a sample's tokens
        _case("norm-sequence-train", "norm", 16, 4096, 512, groups=32, gate=False, over="sequence", grad=True),
        # the same in float32 at odd sizes, groups of 10 channels
        _case("norm-sequence-f32-odd", "norm", 3, 1201, 320, groups=32, gate=False, over="sequence", dtype="f32", grad=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Another case of the same ranges, no larger than the listed ones of its kind."""
    while True:
        c = _draw(rng)
        most = max(_cost(x) for x in listed() if x["op"] == c["op"] and (x["grad"] or not c["grad"]))
        if _cost(c) <= most * (1.0 if c["dtype"] == "bf16" else 0.25):
            return c


def _cost(case):
    return work(case)["flops"] if case["op"] == "scan" else work(case)["bytes"]


def _draw(rng):
    op = rng.choice(("conv", "scan", "scan", "norm"))
    B, T = _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
    dtype = rng.choice(("bf16", "bf16", "f32"))
    few = rng.random() < 0.3
    if few:
        B, T = _log_int(rng, 1, 128), rng.choice((1, 1, 1, rng.randint(2, 16)))
    grad = not few and rng.random() < 0.5
    if op == "conv":
        C = rng.choice((_log_int(rng, 8, 256) * 8, _log_int(rng, 1, 2048)))
        return _case(None, op, B, T, C, K=rng.choice((4, 4, 3, 2)), dtype=dtype, grad=grad, act=rng.choice(("silu", "none")),
                     bias=rng.random() < 0.8, carry=few or rng.random() < 0.4, starts=rng.random() < 0.3,
                     columns=rng.random() < 0.3)
    if op == "scan":
        G = rng.choice((1, 1, 1, 2, 8))
        C = G * rng.choice((_log_int(rng, 1, 2048 // (8 * G)) * 8, _log_int(rng, 1, 2048 // G)))
        return _case(None, op, B, T, C, N=rng.choice((16, 16, 16, 8, 4, 10, 32, 64)), G=G, dtype=dtype, grad=grad,
                     gate=rng.random() < 0.7, skip=rng.random() < 0.8, carry=few or rng.random() < 0.4, starts=rng.random() < 0.3)
    groups = rng.choice((1, 4, 24, 32))
    C = groups * rng.choice((rng.choice((8, 16, 32, 64)), _log_int(rng, 2, max(2, 2048 // groups))))
    return _case(None, op, B, T, C, groups=groups, dtype=dtype, grad=grad, act=rng.choice(("silu", "silu", "gelu", "none")),
                 gate=rng.random() < 0.5, over="token" if few else rng.choice(("token", "sequence")), affine=rng.random() < 0.8)


# ---- what a user's program has in hand ---------------------------------------------------------------------------

LEAVES = {"conv": ("x", "weight", "bias", "state"), "scan": ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state"),
          "norm": ("x", "weight", "bias", "gate")}


def _randn(g, *shape, scale=1.0, at=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + at).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, T, C, dt = case["B"], case["T"], case["C"], DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "conv":
        wide = _randn(g, B, T, C + 64 if case["columns"] else C, dtype=dt)
        s["x"] = wide[..., 32:32 + C] if case["columns"] else wide
        s["weight"] = _randn(g, C, case["K"], scale=case["K"] ** -0.5, dtype=dt)
        s["bias"] = _randn(g, C, scale=0.1, dtype=dt) if case["bias"] else None
        s["state"] = _randn(g, B, case["K"] - 1, C, dtype=dt) if case["carry"] else None
    elif case["op"] == "scan":
        N, G = case["N"], case["G"]
        s["x"] = _randn(g, B, T, C, scale=0.5, dtype=dt)
        s["dt"] = _randn(g, B, T, C, scale=0.5, dtype=dt)
        # decays as such layers start: rates -1 .. -N per channel, steps of 0.001 to 0.1
        s["A"] = -torch.exp(torch.log(torch.arange(1, N + 1, device="cuda")) + _randn(g, C, N, scale=0.1))
        s["B"] = _randn(g, B, T, G, N, dtype=dt)
        s["C"] = _randn(g, B, T, G, N, dtype=dt)
        s["D"] = _randn(g, C, scale=0.1, at=1.0) if case["skip"] else None
        s["z"] = _randn(g, B, T, C, dtype=dt) if case["gate"] else None
        step = torch.exp(torch.rand(C, generator=g, device="cuda") * math.log(100.0) + math.log(0.001))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["state"] = _randn(g, B, C, N, scale=0.1) if case["carry"] else None
        if case["carry"] and case["grad"]:
            s["dstate"] = _randn(g, B, C, N, scale=1e-2)
    else:
        s["x"] = _randn(g, B, T, C, at=0.1, dtype=dt)
        s["weight"] = _randn(g, C, scale=0.1, at=1.0, dtype=dt) if case["affine"] else None
        s["bias"] = _randn(g, C, scale=0.1, dtype=dt) if case["affine"] else None
        s["gate"] = _randn(g, B, T, C, dtype=dt) if case["gate"] else None
    s["starts"] = torch.rand(B, T, generator=g, device="cuda") < 1 / 97 if case.get("starts") else None
    if case["grad"]:
        s["dy"] = _randn(g, B, T, C, scale=1e-2, dtype=dt)
        if case["op"] == "conv" and case["carry"]:
            s["dstate"] = _randn(g, B, case["K"] - 1, C, scale=1e-2, dtype=dt)
        for n in LEAVES[case["op"]]:
            if s[n] is not None:
                s[n] = s[n].detach().requires_grad_()
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(state):
    c = state["case"]
    leaves = [state[n] for n in LEAVES[c["op"]] if state[n] is not None]
    with torch.set_grad_enabled(c["grad"]):
        if own:
            ys = _call(state)
        elif c["op"] == "scan":
            return _scan_plain(state)
        else:
            ys = _conv_plain(state) if c["op"] == "conv" else [_norm_plain(state)]
        if not c["grad"]:
            return ys
        grads = [state["dy"]] + ([state["dstate"]] if "dstate" in state else [])
        return [*ys, *torch.autograd.grad(ys[:len(grads)], leaves, grads)]


def _call(s):
    import ttt_rs_b200 as tb
    c = s["case"]
    act = None if c.get("act") in (None, "none") else c["act"]
    if c["op"] == "conv":
        return list(tb.causal_conv(s["x"], s["weight"], s["bias"], s["state"], activation=act, starts=s["starts"]))
    if c["op"] == "scan":
        return list(tb.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                      state=s["state"], starts=s["starts"]))
    return [tb.group_norm(s["x"], c["groups"], s["weight"], s["bias"], gate=s["gate"], activation=act, eps=1e-5, over=c["over"])]


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _act_plain(v, act):
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":  # (the tanh form)
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _conv_plain(s):
    """Windows of K inputs, the ones before a start left out."""
    c, x = s["case"], s["x"]
    B, T, C, K = c["B"], c["T"], c["C"], c["K"]
    before = x.new_zeros(B, K - 1, C) if s["state"] is None else s["state"]
    rows = torch.cat([before, x], 1)
    doc = torch.zeros(B, T, dtype=torch.long, device=x.device) if s["starts"] is None else s["starts"].long().cumsum(1)
    doc = torch.cat([doc.new_zeros(B, K - 1), doc], 1)
    seen = doc.unfold(1, K, 1) == doc[:, K - 1:, None]  # [B, T, K]
    v = (rows.float().unfold(1, K, 1) * s["weight"].float() * seen[:, :, None]).sum(-1)
    if s["bias"] is not None:
        v = v + s["bias"].float()
    return [_act_plain(v, c["act"]).to(x.dtype), torch.where((doc[:, T:] == doc[:, -1:])[..., None], rows[:, T:], 0.0)]


def _norm_plain(s):
    c = s["case"]
    x = s["x"].float().unflatten(-1, (c["groups"], -1))
    dims = (3,) if c["over"] == "token" else (1, 3)
    x = x - x.mean(dims, keepdim=True)
    n = (x * torch.rsqrt((x * x).mean(dims, keepdim=True) + 1e-5)).flatten(2)
    if c["affine"]:
        n = n * s["weight"].float() + s["bias"].float()
    y = _act_plain(n, c["act"]) if s["gate"] is None else n * _act_plain(s["gate"].float(), c["act"])
    return y.to(s["x"].dtype)


def _along_tokens(a, b):
    """h_t = a_t h_{t-1} + b_t of [B, T, ...], by doubling."""
    n = 1
    while n < a.shape[1]:
        b = torch.cat([b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]], 1)
        a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return b


def _scan_plain(s):
    c = s["case"]
    with torch.no_grad():
        x, v, A = s["x"].float(), s["dt"].float() + s["dt_bias"], s["A"]
        Bm, Cm = (s[n].float().repeat_interleave(c["C"] // c["G"], 2) for n in ("B", "C"))  # [B, T, C, N]
        d = torch.logaddexp(v, torch.zeros_like(v))
        a = torch.exp(d[..., None] * A)
        if s["starts"] is not None:
            a = a.masked_fill(s["starts"][..., None, None], 0.0)
        b = (d * x)[..., None] * Bm
        if s["state"] is not None:
            b[:, 0] += a[:, 0] * s["state"]
        h = _along_tokens(a, b)
        del b
        y = (h * Cm).sum(-1)
        if s["D"] is not None:
            y = y + s["D"] * x
        gate = 1.0 if s["z"] is None else _act_plain(s["z"].float(), "silu")
        out = [(y * gate).to(s["x"].dtype), h[:, -1].clone()]
        if not c["grad"]:
            return out
        return out + _scan_plain_grads(s, x, v, d, a, h, y, gate, Bm, Cm)


def _scan_plain_grads(s, x, v, d, a, h, y, gate, Bm, Cm):
    c, dt = s["case"], s["x"].dtype
    dout = s["dy"].float()
    dy = dout * gate
    dh = dy[..., None] * Cm
    if "dstate" in s:
        dh[:, -1] += s["dstate"]
    dCm = _sum_groups(dy[..., None] * h, c)
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    dh = _along_tokens(after.flip(1), dh.flip(1)).flip(1)
    first = torch.zeros_like(h[:, :1]) if s["state"] is None else s["state"][:, None]
    da = dh * torch.cat([first, h[:, :-1]], 1) * a
    into = (dh * Bm).sum(-1)
    dv = ((da * s["A"]).sum(-1) + into * x) / (1.0 + torch.exp(-v))
    dx = d * into
    if s["D"] is not None:
        dx = dx + s["D"] * dy
    grads = [dx.to(dt), dv.to(dt), (da * d[..., None]).sum((0, 1)), _sum_groups(dh * (d * x)[..., None], c).to(dt), dCm.to(dt)]
    if s["D"] is not None:
        grads.append((dy * x).sum((0, 1)))
    if s["z"] is not None:
        z = s["z"].float()
        sig = 1.0 / (1.0 + torch.exp(-z))
        grads.append((dout * y * sig * (1.0 + z * (1.0 - sig))).to(dt))
    grads.append(dv.sum((0, 1)))
    if s["state"] is not None:
        grads.append(a[:, 0] * dh[:, 0])
    return grads


def _sum_groups(t, c):
    return t.unflatten(2, (c["G"], -1)).sum(3)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    s = {k: (v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v)
         for k, v in prepare(case, seed).items()}
    with torch.no_grad():
        return {"conv": _conv_exact, "scan": _scan_exact, "norm": _norm_exact}[case["op"]](s)


def _act_exact(v, act):
    """The activation and its derivative."""
    if act == "silu":
        g = torch.sigmoid(v)
        return v * g, g + v * g * (1.0 - g)
    if act == "gelu":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (v + 0.044715 * v ** 3))
        return 0.5 * v * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * v * v)
    return v, torch.ones_like(v)


def _conv_exact(s):
    """Tap by tap: the input `back` tokens before, where none of the tokens since is a start."""
    c, x, w = s["case"], s["x"], s["weight"]
    B, T, C, K = c["B"], c["T"], c["C"], c["K"]
    rows = torch.cat([torch.zeros(B, K - 1, C, dtype=x.dtype, device=x.device) if s["state"] is None else s["state"], x], 1)
    cut = torch.zeros(B, T, dtype=torch.bool, device=x.device) if s["starts"] is None else s["starts"]
    cut = torch.nn.functional.pad(cut, (K - 1, 0))
    reach, open_ = [], torch.ones(B, T, dtype=torch.bool, device=x.device)
    for back in range(K):
        reach.append(open_[..., None].double())
        open_ = open_ & ~cut[:, K - 1 - back:K - 1 - back + T]
    v = torch.zeros_like(x) + (0.0 if s["bias"] is None else s["bias"])
    for back in range(K):
        v = v + reach[back] * rows[:, K - 1 - back:K - 1 - back + T] * w[:, K - 1 - back]
    y, slope = _act_exact(v, c["act"])
    tail, keep = rows[:, T:].clone(), torch.ones(B, 1, dtype=torch.double, device=x.device)
    kept = []
    for i in reversed(range(K - 1)):  # a start hides what lies before it
        kept.append(keep)
        tail[:, i] *= keep
        keep = keep * ~cut[:, T + i, None]
    if not c["grad"]:
        return [y, tail]
    dv = s["dy"] * slope
    drows, dw = torch.zeros_like(rows), torch.zeros_like(w)
    for back in range(K):
        at = slice(K - 1 - back, K - 1 - back + T)
        drows[:, at] += reach[back] * dv * w[:, K - 1 - back]
        dw[:, K - 1 - back] = (reach[back] * dv * rows[:, at]).sum((0, 1))
    if "dstate" in s:
        for i, k in zip(reversed(range(K - 1)), kept):
            drows[:, T + i] += k * s["dstate"][:, i]
    out = [y, tail, drows[:, K - 1:], dw]
    if s["bias"] is not None:
        out.append(dv.sum((0, 1)))
    return out + ([drows[:, :K - 1]] if s["state"] is not None else [])


def _norm_exact(s):
    c, x = s["case"], s["x"]
    g, dims = c["groups"], (-1,) if c["over"] == "token" else (1, -1)
    w = s["weight"] if c["affine"] else torch.ones_like(x[0, 0])
    b = s["bias"] if c["affine"] else torch.zeros_like(x[0, 0])
    xg = x.unflatten(-1, (g, -1))
    var, mean = torch.var_mean(xg, dims, correction=0, keepdim=True)
    r = 1.0 / torch.sqrt(var + 1e-5)
    n = ((xg - mean) * r).flatten(2)
    u = n * w + b
    gate = s["gate"]
    act, slope = _act_exact(u if gate is None else gate, c["act"])
    out = [act if gate is None else u * act]
    if not c["grad"]:
        return out
    du = s["dy"] * (slope if gate is None else act)
    p = (du * w).unflatten(-1, (g, -1))
    ng = n.unflatten(-1, (g, -1))
    out.append((r * (p - p.mean(dims, keepdim=True) - ng * (p * ng).mean(dims, keepdim=True))).flatten(2))
    if c["affine"]:
        out += [(du * n).sum((0, 1)), du.sum((0, 1))]
    return out + ([s["dy"] * u * slope] if gate is not None else [])


def _scan_exact(s):
    """Token by token."""
    c, x, A = s["case"], s["x"], s["A"]
    B, T, C, N, each = c["B"], c["T"], c["C"], c["N"], c["C"] // c["G"]
    opt = dict(dtype=torch.float64, device=x.device)
    v = s["dt"] + s["dt_bias"]
    d = torch.where(v > 0, v, 0.0) + torch.log1p(torch.exp(-v.abs()))
    keep = torch.ones(B, T, 1, 1, **opt) if s["starts"] is None else (~s["starts"])[:, :, None, None].double()
    h = torch.zeros(B, C, N, **opt) if s["state"] is None else s["state"]
    saved, y = [h], torch.empty(B, T, C, **opt)
    for t in range(T):
        Bt, Ct = (s[n][:, t, :, None].expand(B, c["G"], each, N).reshape(B, C, N) for n in ("B", "C"))
        h = torch.exp(d[:, t, :, None] * A) * keep[:, t] * h + (d[:, t] * x[:, t])[..., None] * Bt
        y[:, t] = torch.einsum("bcn,bcn->bc", h, Ct)
        if c["grad"]:
            saved.append(h)
    skip = s["D"] if s["D"] is not None else torch.zeros(C, **opt)
    y += skip * x
    gate, slope = (1.0, 0.0) if s["z"] is None else _act_exact(s["z"], "silu")
    if not c["grad"]:
        return [y * gate, h]
    dy = s["dy"] * gate
    dh = s["dstate"] if "dstate" in s else torch.zeros(B, C, N, **opt)
    dx, dd, dA = skip * dy, torch.empty_like(d), torch.zeros_like(A)
    dB, dC = torch.empty_like(s["B"]), torch.empty_like(s["C"])
    for t in reversed(range(T)):
        Bt, Ct = (s[n][:, t, :, None].expand(B, c["G"], each, N).reshape(B, C, N) for n in ("B", "C"))
        dh = dh + dy[:, t, :, None] * Ct
        dC[:, t] = (dy[:, t, :, None] * saved[t + 1]).unflatten(1, (c["G"], each)).sum(2)
        dB[:, t] = (dh * (d[:, t] * x[:, t])[..., None]).unflatten(1, (c["G"], each)).sum(2)
        into = (dh * Bt).sum(-1)
        dh = dh * torch.exp(d[:, t, :, None] * A) * keep[:, t]
        way = dh * saved[t]
        dA += (way * d[:, t, :, None]).sum(0)
        dd[:, t] = (way * A).sum(-1) + into * x[:, t]
        dx[:, t] += into * d[:, t]
    dv = dd * torch.sigmoid(v)
    out = [y * gate, h, dx, dv, dA, dB, dC]
    if s["D"] is not None:
        out.append((dy * x).sum((0, 1)))
    if s["z"] is not None:
        out.append(s["dy"] * y * slope)
    out.append(dv.sum((0, 1)))
    return out + ([dh] if s["state"] is not None else [])


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    B, T, C = case["B"], case["T"], case["C"]
    es, n = 2 if case["dtype"] == "bf16" else 4, B * T * C
    mask = B * T if case.get("starts") else 0
    if case["op"] == "conv":
        K = case["K"]
        tail = B * (K - 1) * C * es * (2 if case["carry"] else 1)
        b = 2 * n * es + tail + mask + C * (K + 1) * es
        f = n * (2 * K + 5)
        if case["grad"]:  # x and the result's gradient in, the input's gradient out
            b += 3 * n * es + tail + mask + 2 * C * (K + 1) * es
            f += n * (6 * K + 12)
        return {"bytes": b, "flops": f}
    if case["op"] == "scan":
        N, bc = case["N"], B * T * case["G"] * case["N"] * es
        wide, z = 2 + bool(case["gate"]), bool(case["gate"])  # x, dt, z
        params, state = 4 * C * (N + 2), 4 * B * C * N
        b = (wide + 1) * n * es + 2 * bc + mask + params + state * (2 if case["carry"] else 1)
        f = n * N * 8 + n * 12
        if case["grad"]:
            b += (2 * wide + 1) * n * es + 4 * bc + mask + 2 * params + state * (3 if case["carry"] else 0)
            f += n * N * 24 + n * 20
        return {"bytes": b, "flops": f}
    wide = 1 + bool(case["gate"])
    b, f = (wide + 1) * n * es + 2 * C * es, n * 12
    if case["grad"]:
        b += (2 * wide + 1) * n * es + 4 * C * es
        f += n * 24
    return {"bytes": b, "flops": f}
