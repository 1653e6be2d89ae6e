"""Performance cases of the operators beside the TTT inner loops: what a layer that norms and rotates its queries and keys
and remembers through a gated linear recurrence has its users run.

A case is a dict of plain values; its "op" says which operator it is a call of:

    rotary     rotary positions on [B, H, T, F]: neighbouring or half-split pairs, the whole head or its first features,
               angles scaled for long contexts; forward, or forward + backward
    qk_norm    root-mean-square norm of every head's query and key with its weight, and the rotation, in one pass
    gated      W_t = exp(g_t) W_{t-1} + beta_t k_t^T v_t,  o_t = q_t W_t for every (batch, head) stream: whole sequences,
               forward or forward + backward, and steps of a few tokens against the resident state

`run` computes a case in elementary torch operations, or through the framework's entry points where `own` is set.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BASE = {"dtype": "bf16", "F": 64, "grad": False, "start": 0}
ROT = {"rdim": 64, "pairs": "interleaved", "scaling": "none", "factor": 1.0, "orig": 0, "theta": 10000.0, "wrap": 0,
       "layout": "heads", "ragged": False}
GATED = {"resets": False, "carry": False, "beta": True}


def _case(name, op, B, H, T, **more):
    c = dict(BASE, **(GATED if op == "gated" else ROT), op=op, B=B, H=H, T=T)
    c.update(more)
    if op == "qk_norm":
        c.setdefault("Hk", H)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # a generated token of a small batch: the call a serving loop repeats for each layer and token
        _case("gated-token-b8", "gated", 8, 12, 1),
        # a generated token of a large batch, 2048 resident states
        _case("gated-token-b128", "gated", 128, 16, 1),
        # a few prompts of odd length, no gradients: time to the first token
        _case("gated-prompt-odd", "gated", 3, 12, 1201),
        # one very long prompt: fewer streams than the card has processors
        _case("gated-prompt-long", "gated", 1, 12, 32768),
        # training at the 125M layer shape: the headline workload's sizes
        _case("gated-train-b32", "gated", 32, 12, 2048, grad=True),
        # training on one long sequence, the state and its gradient carried from chunk to chunk, documents packed one behind
        # the other (a decay of zero at their starts)
        _case("gated-train-long", "gated", 1, 16, 8192, grad=True, resets=True, carry=True),
        # float32 (parity and debugging runs), heads of 32 features, an odd length
        _case("gated-train-f32-d32", "gated", 2, 24, 515, F=32, dtype="f32", grad=True),
        # the position of one generated token of a small batch, deep in its context
        _case("rotary-token-b8", "rotary", 8, 12, 1, start=32767, pairs="half"),
        # a long prompt, angles scaled by parts from 4096 positions to eight times as many
        _case("rotary-prompt-long", "rotary", 1, 32, 32768, pairs="half", scaling="by_parts", factor=8.0, orig=4096,
              layout="tokens"),
        # training in float32 with a part of an 80-wide head rotated, positions of sequences that are padded on the left
        _case("rotary-train-part-f32", "rotary", 5, 7, 1001, F=80, rdim=24, dtype="f32", grad=True, ragged=True),
        # a generated token, queries and keys as column blocks of the projection, fewer heads of keys than of queries
        _case("qk-norm-token-b8", "qk_norm", 8, 12, 1, Hk=4, start=1000, layout="projection"),
        # training at the 125M layer shape, columns of the projection in, the inner loop's [B, H, T, F] out, positions
        # wrapped at the mini-batch as the layer has them
        _case("qk-norm-train-b32", "qk_norm", 32, 12, 2048, grad=True, wrap=16, layout="projection"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Another case of the same ranges, no larger than the listed ones of its kind."""
    while True:
        c = _draw(rng)
        most = max(_cost(x) for x in listed() if x["op"] == c["op"])
        if _cost(c) <= most * (1.0 if c["dtype"] == "bf16" else 0.25):
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _draw(rng):
    op = rng.choice(("rotary", "qk_norm", "gated", "gated"))
    B, H, T = _log_int(rng, 1, 64), _log_int(rng, 1, 32), _log_int(rng, 1, 32768)
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if op == "gated":
        step = rng.random() < 0.3
        if step:
            B, T = _log_int(rng, 1, 128), rng.choice((1, 1, 1, rng.randint(2, 16)))
        return _case(None, op, B, H, T, F=rng.choice((64, 64, 32)), dtype=dtype, grad=not step and rng.random() < 0.5,
                     resets=rng.random() < 0.3, carry=rng.random() < 0.4, beta=rng.random() < 0.8)
    if rng.random() < 0.25:
        T = 1
    F = rng.choice((64, 64, 32, 128, 96, 80, 256))
    scaling = rng.choice(("none", "none", "linear", "ntk", "by_parts"))
    more = dict(F=F, rdim=rng.choice((F, F, F // 2, F // 4)), dtype=dtype, grad=T > 1 and rng.random() < 0.5,
                pairs=rng.choice(("interleaved", "half")), scaling=scaling, start=rng.choice((0, rng.randint(0, 1 << 20))),
                factor=1.0 if scaling == "none" else rng.choice((2.0, 8.0, 32.0)), orig=rng.choice((2048, 8192)),
                theta=rng.choice((10000.0, 500000.0)), wrap=rng.choice((0, 0, 16)),
                layout=rng.choice(("heads", "tokens", "projection")), ragged=rng.random() < 0.3)
    if op == "qk_norm":
        more["Hk"] = rng.choice([h for h in (H, H, max(1, H // 2), 1) if H % h == 0])
    return _case(None, op, B, H, T, **more)


# ---- what a user's program has in hand ---------------------------------------------------------------------------

def _randn(g, *shape, scale=1.0, at=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + at).to(dtype)


def _positions(case, g):
    """Positions [B, T] of sequences padded on the left (the padding counts up to zero), or None: start + t."""
    if not case["ragged"]:
        return None
    B, T = case["B"], case["T"]
    pad = torch.randint(0, T // 2 + 1, (B, 1), generator=g, device="cuda")
    return (torch.arange(T, device="cuda") - pad + case["start"]).clamp_min(0)


def _heads(g, case, heads, buf, col):
    """[B, H, T, F] values as the case lays them out: of their own, [B, T, H, F] turned, or columns of a projection."""
    B, T, F, dt = case["B"], case["T"], case["F"], DTYPES[case["dtype"]]
    if case["layout"] == "heads":
        return _randn(g, B, heads, T, F, dtype=dt)
    if case["layout"] == "tokens":
        return _randn(g, B, T, heads, F, dtype=dt).transpose(1, 2)
    return buf[..., col:col + heads * F].unflatten(-1, (heads, F)).transpose(1, 2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, T, F, dt = case["B"], case["H"], case["T"], case["F"], DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "gated":
        # rows and learning rates as the layer makes them; a head forgets up to 2^-1 .. 2^-7 of its state per token
        for n in ("q", "k", "v"):
            s[n] = _randn(g, B, H, T, F, scale=F ** -0.5, dtype=dt)
        gate = torch.sigmoid(_randn(g, B, H, T))
        most = 2.0 ** -(1 + 6 * torch.arange(H, device="cuda") / H)
        s["decay"] = torch.log1p(-most[:, None] * gate)
        s["beta"] = gate if case["beta"] else None
        if case["resets"]:
            start = torch.rand(B, 1, T, generator=g, device="cuda") < 1 / 257
            s["decay"] = s["decay"].masked_fill(start, -math.inf)
        s["state"] = _randn(g, B, H, F, F, scale=0.02)
        if case["grad"]:
            s["dout"] = _randn(g, B, H, T, F, scale=1e-2, dtype=dt)
            s["dstate"] = _randn(g, B, H, F, F, scale=1e-2) if case["carry"] else None
    else:
        Hk = case.get("Hk", 0)
        buf = None
        if case["layout"] == "projection":
            buf = _randn(g, B, T, (H + 2 * Hk) * F + 16, dtype=dt)
        s["q"] = _heads(g, case, H, buf, 0)
        if case["op"] == "qk_norm":
            s["k"] = _heads(g, case, Hk, buf, H * F)
            s["wq"] = _randn(g, F, scale=0.1, at=1.0, dtype=dt)
            s["wk"] = _randn(g, F, scale=0.1, at=1.0, dtype=dt)
        s["pos"] = _positions(case, g)
        if case["grad"]:
            s["dq"] = _randn(g, B, H, T, F, scale=1e-2, dtype=dt)
            if case["op"] == "qk_norm":
                s["dk"] = _randn(g, B, Hk, T, F, scale=1e-2, dtype=dt)
    if case["grad"]:
        for n in ("q", "k", "v", "decay", "beta", "state", "wq", "wk"):
            if s.get(n) is not None:
                s[n] = s[n].detach().requires_grad_()
    if own and case["op"] != "gated":
        import ttt_rs_b200 as tb
        s["rot"] = tb.Rotary(tb.RotaryConfig(
            head_dim=F, rotary_dim=case["rdim"], theta=case["theta"], layout=case["pairs"], scaling=case["scaling"],
            factor=case["factor"], original_length=case["orig"], wrap=case["wrap"]), device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(state):
    op, grad = state["case"]["op"], state["case"]["grad"]
    with torch.set_grad_enabled(grad):
        if op == "gated":
            return _run_gated(state)
        if op == "rotary":
            y = _call_rotary(state)
            return [y, *torch.autograd.grad(y, state["q"], state["dq"])] if grad else [y]
        ys = list(_call_qk_norm(state))
        if not grad:
            return ys
        leaves = [state[n] for n in ("q", "k", "wq", "wk")]
        return ys + list(torch.autograd.grad(ys, leaves, [state["dq"], state["dk"]]))


def _run_gated(s):
    args = [s[n] for n in ("q", "k", "v", "decay", "beta", "state")]
    if own:
        import ttt_rs_b200 as tb
        out, new = tb.fused_gated_linear(*args)
    else:
        out, new = _gated_plain(*args)
    if not s["case"]["grad"]:
        return [out, new]
    leaves = [a for a in args if a is not None]
    if s["dstate"] is None:
        return [out, new, *torch.autograd.grad(out, leaves, s["dout"])]
    return [out, new, *torch.autograd.grad([out, new], leaves, [s["dout"], s["dstate"]])]


def _call_rotary(s):
    c = s["case"]
    if own:
        import ttt_rs_b200 as tb
        return tb.rotary(s["q"], s["rot"], start_idx=c["start"], positions=s["pos"])
    return _rotate_plain(s["q"].float(), c, s["pos"]).to(s["q"].dtype)


def _call_qk_norm(s):
    c = s["case"]
    if own:
        import ttt_rs_b200 as tb
        return tb.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["rot"], eps=1e-6, start_idx=c["start"],
                                 positions=s["pos"])
    return [_rotate_plain(_norm_plain(x, w), c, s["pos"]).to(x.dtype) for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"]))]


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _norm_plain(x, w):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()


def _rotate_plain(x, c, pos):
    r, i = c["rdim"], torch.arange(c["rdim"] // 2, device="cuda", dtype=torch.float64)
    theta = c["theta"] * (c["factor"] ** (r / (r - 2)) if c["scaling"] == "ntk" else 1.0)
    freq = theta ** (-2.0 * i / r)
    size = 1.0
    if c["scaling"] == "linear":
        freq = freq / c["factor"]
    elif c["scaling"] == "by_parts":
        ramp = ((c["orig"] * freq / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        freq = freq * (ramp + (1.0 - ramp) / c["factor"])
        size = 0.1 * math.log(c["factor"]) + 1.0
    if pos is None:
        pos = (torch.arange(c["T"], device="cuda") + c["start"])[None]
    if c["wrap"]:
        pos = pos % c["wrap"]
    angle = (pos[..., None].double() * freq)[:, None]  # [B or 1, 1, T, r / 2]
    cos, sin = (torch.cos(angle) * size).float(), (torch.sin(angle) * size).float()
    if c["pairs"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _gated_plain(q, k, v, decay, beta, state, chunk=64):
    """Chunk by chunk: inside a chunk the products of queries and keys under their decays, between chunks the state.  A decay
    of zero (g = -inf) is one of exp(-2000): in 64 bits the sums of logarithms that differences are taken of lose nothing."""
    dt, T = q.dtype, q.shape[2]
    q, k, v = q.float(), k.float(), v.float()
    g = decay.double().clamp_min(-2000.0)
    w, outs = state, []
    for t0 in range(0, T, chunk):
        at = slice(t0, min(T, t0 + chunk))
        qc, kc, vc = q[:, :, at], k[:, :, at], v[:, :, at]
        cum = g[:, :, at].cumsum(-1)
        n = cum.shape[-1]
        upper = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        near = (cum[..., :, None] - cum[..., None, :]).masked_fill(upper, -2000.0).exp().float()
        last = (cum[..., -1:] - cum).exp().float()
        if beta is not None:
            near, last = near * beta[:, :, None, at], last * beta[:, :, at]
        out = (qc @ kc.transpose(-1, -2) * near) @ vc + cum.exp().float()[..., None] * (qc @ w)
        w = cum[..., -1, None, None].exp().float() * w + (kc * last[..., None]).transpose(-1, -2) @ vc
        outs.append(out)
    return torch.cat(outs, 2).to(dt), w


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    s = {k: (v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v)
         for k, v in prepare(case, seed).items()}
    with torch.no_grad():
        if case["op"] == "gated":
            return _gated_exact(s)
        z = _phasors(case, s["pos"])
        if case["op"] == "rotary":
            y = [_turn(s["q"], z, case)]
            return y + [_turn(s["dq"], z.conj(), case)] if case["grad"] else y
        ys, grads, wgrads = [], [], []
        for x, w, d in ((s["q"], s["wq"], s.get("dq")), (s["k"], s["wk"], s.get("dk"))):
            r = 1.0 / torch.sqrt(x.square().sum(-1, keepdim=True) / case["F"] + 1e-6)
            ys.append(_turn(x * r * w, z, case))
            if case["grad"]:
                u = _turn(d, z.conj(), case)
                wgrads.append((u * x * r).sum((0, 1, 2)))
                grads.append(r * u * w - x * r ** 3 * (u * w * x).sum(-1, keepdim=True) / case["F"])
        return ys + grads + wgrads


def _phasors(c, pos):
    """exp(i angle) times the size of the scaled rotation, [B or 1, 1, T, rdim / 2]."""
    r, freqs, size = c["rdim"], [], 1.0
    for i in range(r // 2):
        f = c["theta"] ** (-2.0 * i / r)
        if c["scaling"] == "ntk":
            f = (c["theta"] * c["factor"] ** (r / (r - 2))) ** (-2.0 * i / r)
        elif c["scaling"] == "linear":
            f /= c["factor"]
        elif c["scaling"] == "by_parts":
            keep = min(1.0, max(0.0, (c["orig"] * f / (2 * math.pi) - 1.0) / 31.0))
            f = keep * f + (1.0 - keep) * f / c["factor"]
            size = 1.0 + 0.1 * math.log(c["factor"])
        freqs.append(f)
    if pos is None:
        pos = torch.arange(c["start"], c["start"] + c["T"], device="cuda").reshape(1, -1)
    pos = pos.remainder(c["wrap"]) if c["wrap"] else pos
    angle = pos.double().reshape(pos.shape[0], 1, pos.shape[1], 1) * torch.tensor(freqs, dtype=torch.float64, device="cuda")
    return torch.polar(torch.full_like(angle, size), angle)


def _turn(x, z, c):
    r, y = c["rdim"], x.clone(memory_format=torch.contiguous_format)
    one, two = ((slice(0, r // 2), slice(r // 2, r)) if c["pairs"] == "half" else (slice(0, r, 2), slice(1, r, 2)))
    t = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * z
    y[..., one], y[..., two] = t.real, t.imag
    return y


def _gated_exact(s):
    """Token by token.  The gradient of g_t is a_t <dW_t, W_{t-1}>: with P_t = <dW_t, W_t> it is P_t less what token t itself
    wrote, and P_{t-1} is that plus what token t - 1 read."""
    c = s["case"]
    q, k, v, g, w = (s[n] for n in ("q", "k", "v", "decay", "state"))
    beta = s["beta"] if s["beta"] is not None else torch.ones_like(g)
    a, T = g.exp(), c["T"]
    out, dq = torch.empty_like(q), torch.empty_like(q)
    for t in range(T):
        w = a[:, :, t, None, None] * w + (beta[:, :, t, None] * k[:, :, t])[..., None] * v[:, :, t, None, :]
        out[:, :, t] = torch.einsum("bhk,bhkv->bhv", q[:, :, t], w)
        if c["grad"]:
            dq[:, :, t] = torch.einsum("bhkv,bhv->bhk", w, s["dout"][:, :, t])
    if not c["grad"]:
        return [out, w]
    dk, dv, dg, dbeta = torch.empty_like(k), torch.empty_like(v), torch.empty_like(g), torch.empty_like(g)
    dw = torch.zeros_like(w) if s["dstate"] is None else s["dstate"].clone()
    p = (dw * w).sum((-1, -2))
    for t in reversed(range(T)):
        dw = dw + q[:, :, t, :, None] * s["dout"][:, :, t, None, :]
        p = p + (q[:, :, t] * dq[:, :, t]).sum(-1)
        u = torch.einsum("bhkv,bhv->bhk", dw, v[:, :, t])
        dk[:, :, t] = beta[:, :, t, None] * u
        dv[:, :, t] = beta[:, :, t, None] * torch.einsum("bhkv,bhk->bhv", dw, k[:, :, t])
        dbeta[:, :, t] = (u * k[:, :, t]).sum(-1)
        p = p - beta[:, :, t] * dbeta[:, :, t]
        p = torch.where(a[:, :, t] == 0, 0.0, p)
        dg[:, :, t] = p
        dw = a[:, :, t, None, None] * dw
    return [out, w, dq, dk, dv, dg] + ([dbeta] if s["beta"] is not None else []) + [dw]


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    B, H, T, F = case["B"], case["H"], case["T"], case["F"]
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "gated":
        n = B * H * T
        gates = 4 * n * (2 if case["beta"] else 1)
        state = 4 * B * H * F * F
        b = 4 * n * F * es + gates + 2 * state
        f = n * F * F * 5  # state update (multiply, add, decay), output (multiply, add)
        if case["grad"]:
            b += 7 * n * F * es + 2 * gates + (3 if case["carry"] else 2) * state
            f += n * F * F * 15  # W again, dW, and its or W's product with q, k, v and d out
        return {"bytes": b, "flops": f}
    rows = B * T * (H + case.get("Hk", 0))
    per = 2 * F * es
    flops = rows * (3 * case["rdim"] + (4 * F if case["op"] == "qk_norm" else 0))
    if case["grad"]:
        per += (3 if case["op"] == "qk_norm" else 2) * F * es
        flops *= 3
    return {"bytes": rows * per + (B * T * 8 if case["ragged"] else 0), "flops": flops}
