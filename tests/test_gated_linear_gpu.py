"""Gated linear recurrence on the GPU against the token-by-token oracle in float64.

Bounds.  Every result is a sum of products; `mag` is the sum of their absolute values (the oracle on absolute inputs), so a
relative error e of one factor moves a result by at most e mag.  A rounding to bf16 is off by 2^-8 at most.  bf16 inputs:
  o   three roundings (the decayed products q k, the state as the operand of q W, the result)      3 * 2^-8
  dq  two (the decayed products u v, the result)                                                   2 * 2^-8
  dk  two, dv three (also the state's gradient as an operand)                                      2, 3 * 2^-8
  float32 results (state, gradients of gates and of the state): two planes, 2^-16 of a factor at most, no more than two such
  factors in a term, and float32 sums: of up to 64 + 64 terms on the tensor cores, which truncate (2^-23 each, on average half
  of it and of both signs), and of the chunks: 2^-15 + 2^-15
float32 inputs: three planes (2^-23), the same sums: 2^-15.  Exponentials and sums of logarithms: below 2^-20, in the slack."""

import itertools
import math

import pytest
import torch

from oracle import gated_oracle as O

pytestmark = pytest.mark.gpu
NAMES = ("output", "weight_out", "grad_xq", "grad_xk", "grad_xv", "grad_log_decay", "grad_beta", "grad_weight")
BF16 = {"output": 3 * 2 ** -8, "grad_xq": 2 * 2 ** -8, "grad_xk": 2 * 2 ** -8, "grad_xv": 3 * 2 ** -8}
F32 = 2 ** -14


def make(B, H, T, F, dtype, seed=0, beta=True, state=True, resets=False, strong=False):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = (rn(B, H, T, F).to(dtype) for _ in range(3))
    decay = -torch.rand(B, H, T, generator=g) * (20.0 if strong else 0.3)
    if resets:
        decay = decay.masked_fill(torch.rand(B, H, T, generator=g) < 0.1, -math.inf)
    b = torch.rand(B, H, T, generator=g) if beta else None
    w = rn(B, H, F, F) if state else None
    return [q, k, v, decay, b, w], rn(B, H, T, F).to(dtype), rn(B, H, F, F)


def check(got, want, mag, dtype, names=NAMES):
    for name, x, y, m in zip(names, got, want, mag):
        if y is None:
            assert x is None
            continue
        tol = BF16.get(name, F32) if dtype == torch.bfloat16 else F32
        x = x.detach().double().cpu()
        assert x.shape == y.shape and torch.isfinite(x).all(), name
        over = (x - y).abs() - tol * m - 2 ** -120
        assert over.max() <= 0, f"{name}: off by {(x - y).abs().max():.3g} at {int(over.argmax())}, {over.max():.3g} over the bound"


def run(ins, d_out=None, d_w=None, move=lambda t: t):
    import ttt_rs_b200 as tb
    dev = [None if t is None else move(t.cuda()) for t in ins]
    if d_out is None:
        with torch.no_grad():
            return list(tb.fused_gated_linear(*dev))
    dev = [None if t is None else t.detach().requires_grad_() for t in dev]
    out, w = tb.fused_gated_linear(*dev)
    have = [t for t in dev if t is not None]
    grads = iter(torch.autograd.grad([out, w] if d_w is not None else [out], have,
                                     [d_out.cuda(), d_w.cuda()] if d_w is not None else [d_out.cuda()]))
    return [out, w] + [None if t is None else next(grads) for t in dev]


def f64(ins):
    return [None if t is None else t.double() for t in ins]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("F", [64, 32])
@pytest.mark.parametrize("T", [1, 2, 16, 17, 63, 64, 65, 128, 200])
def test_forward(T, F, dtype):
    ins, _, _ = make(2, 3, T, F, dtype, seed=T)
    check(run(ins), O.gated_forward(*f64(ins)), O.gated_magnitudes(*f64(ins)), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("F", [64, 32])
@pytest.mark.parametrize("T", [1, 5, 64, 65, 150])
def test_gradients(T, F, dtype):
    ins, d_out, d_w = make(1, 3, T, F, dtype, seed=T + 1)
    check(run(ins, d_out, d_w), O.gated_grads(*f64(ins), d_out.double(), d_w.double()),
          O.gated_magnitudes(*f64(ins), d_out.double(), d_w.double()), dtype)


@pytest.mark.parametrize("beta,state,dstate", list(itertools.product((True, False), repeat=3)))
def test_optional_inputs(beta, state, dstate):
    ins, d_out, d_w = make(1, 2, 70, 64, torch.bfloat16, beta=beta, state=state)
    dw = d_w if dstate else None
    args = (*f64(ins), d_out.double(), None if dw is None else dw.double())
    check(run(ins, d_out, dw), O.gated_grads(*args), O.gated_magnitudes(*args), torch.bfloat16)
    check(run(ins), O.gated_forward(*f64(ins)), O.gated_magnitudes(*f64(ins)), torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("resets,strong", [(True, False), (True, True), (False, True)])
def test_decays_of_zero_and_strong_ones(resets, strong, dtype):
    """-inf forgets exactly; what stands before it gets no gradient from behind it."""
    ins, d_out, d_w = make(2, 2, 190, 64, dtype, resets=resets, strong=strong, seed=3)
    want = O.gated_grads(*f64(ins), d_out.double(), d_w.double())
    want[5] = want[5].nan_to_num(0.0)
    got = run(ins, d_out, d_w)
    check(got, want, [None if t is None else t.nan_to_num(0.0) for t in O.gated_magnitudes(*f64(ins), d_out.double(), d_w.double())],
          dtype)
    if resets:
        assert (got[5].cpu()[ins[3] == -math.inf] == 0).all()
    check(run(ins)[:2], want, O.gated_magnitudes(*f64(ins)), dtype)


@pytest.mark.parametrize("T", [1200, 1990])
def test_few_streams_in_segments(T):
    """One stream is cut into segments; a call of many streams is not: the same results."""
    ins, d_out, d_w = make(1, 1, T, 64, torch.bfloat16, seed=9, resets=True)
    args = (*f64(ins), d_out.double(), d_w.double())
    want, mag = O.gated_grads(*args), O.gated_magnitudes(*args)
    want[5], mag[5] = want[5].nan_to_num(0.0), mag[5].nan_to_num(0.0)
    check(run(ins, d_out, d_w), want, mag, torch.bfloat16)
    check(run(ins)[:2], want, mag, torch.bfloat16)
    many = [t.expand(160, *t.shape[1:]).contiguous() for t in ins]
    for x, y, name in zip(run(many), want, NAMES):
        check([x[:1], ], [y], [mag[NAMES.index(name)]], torch.bfloat16, [name])
        assert all(torch.equal(x[0], x[i]) for i in (1, 77, 159))


@pytest.mark.parametrize("B,H,T,F,dtype", [(41, 11, 200, 64, torch.bfloat16), (30, 10, 65, 32, torch.bfloat16), (17, 9, 130, 64, torch.float32),
                                           (149, 1, 10, 32, torch.float32), (99, 9, 70, 64, torch.bfloat16)])
def test_more_streams_than_resident_blocks(B, H, T, F, dtype):
    """Streams cut into ranges, a stream's state handed from one block to the next."""
    ins, d_out, d_w = make(B, H, T, F, dtype, seed=B)
    args = (*f64(ins), d_out.double(), d_w.double())
    want, mag = O.gated_grads(*args), O.gated_magnitudes(*args)
    got = run(ins, d_out, d_w)
    check(got, want, mag, dtype)
    check(run(ins)[:2], want, mag, dtype)
    assert all(torch.equal(x, y) for x, y in zip(got, run(ins, d_out, d_w)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_inputs(dtype):
    """[B,T,H,F] turned, columns of a projection, rows that cannot be read in place, expanded gradients."""
    import ttt_rs_b200 as tb
    ins, d_out, _ = make(2, 3, 75, 64, dtype, seed=4)
    want = run(ins, d_out)
    turned = run(ins, d_out, move=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2) if t.dim() == 4 and t.shape[2] == 75 else t)
    buf = torch.zeros(2, 75, 3 * 3 * 64 + 8, dtype=dtype, device="cuda")
    cols = []
    for i in range(3):
        c = buf[..., 192 * i:192 * (i + 1)].unflatten(-1, (3, 64)).transpose(1, 2)
        c.copy_(ins[i])
        cols.append(c)
    odd = torch.zeros(2, 3, 75, 68, dtype=dtype, device="cuda")[..., 1:65]
    odd.copy_(ins[0])
    rest = [t.cuda() for t in ins[3:]]
    with torch.no_grad():
        for q in (cols[0], odd):
            o, w = tb.fused_gated_linear(q, cols[1], cols[2], *rest)
            assert torch.equal(o, want[0]) and torch.equal(w, want[1])
    for x, y in zip(turned, want):
        assert torch.equal(x, y)
    dev = [t.cuda().requires_grad_() for t in ins]
    out, _ = tb.fused_gated_linear(*dev)
    a = torch.autograd.grad(out.sum(), dev, retain_graph=True)
    b = torch.autograd.grad(out, dev, torch.ones_like(out))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_nothing_behind_the_sequence_is_read():
    """What lies behind the last token, and between the rows of a strided tensor, is NaN."""
    import ttt_rs_b200 as tb
    ins, d_out, _ = make(2, 2, 70, 64, torch.bfloat16, seed=5)
    want = run(ins)
    wide = []
    for t in ins[:3]:
        x = torch.full((2, 2, 80, 64), math.nan, dtype=t.dtype, device="cuda")
        x[:, :, :70] = t.cuda()
        wide.append(x[:, :, :70])
    with torch.no_grad():
        got = tb.fused_gated_linear(*wide, *[t.cuda() for t in ins[3:]])
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_carrying_the_state_from_call_to_call():
    """Two calls, the state and its gradient handed on, are one; a step per token is a call of all."""
    import ttt_rs_b200 as tb
    ins, d_out, _ = make(2, 2, 100, 64, torch.float32, seed=6)
    args = (*f64(ins), d_out.double())
    want, mag = O.gated_grads(*args), O.gated_magnitudes(*args)
    dev = [t.cuda().requires_grad_() for t in ins]
    q, k, v, g, b, w = dev
    o1, w1 = tb.fused_gated_linear(q[:, :, :37], k[:, :, :37], v[:, :, :37], g[..., :37], b[..., :37], w)
    o2, w2 = tb.fused_gated_linear(q[:, :, 37:], k[:, :, 37:], v[:, :, 37:], g[..., 37:], b[..., 37:], w1)
    out = torch.cat([o1, o2], 2)
    grads = torch.autograd.grad(out, dev, d_out.cuda())
    check([out, w2, *grads], want, mag, torch.float32)
    with torch.no_grad():
        state, outs = w, []
        for t in range(20):
            at = slice(t, t + 1)
            o, state = tb.fused_gated_linear(q[:, :, at], k[:, :, at], v[:, :, at], g[..., at], b[..., at], state)
            outs.append(o)
    check([torch.cat(outs, 2)], [want[0][:, :, :20]], [mag[0][:, :, :20]], torch.float32)


def test_gradient_against_differences():
    """float32: <gradient, d> against (f(x + h d) - f(x - h d)) / 2h along a random direction of every input.  f is a polynomial
    in all but g; its third derivative along d is bounded by the value's own size, so that h = 2^-6 leaves h^2 ~ 2^-12 of the
    magnitude, and the results' roundings 2^-18 / 2h."""
    import ttt_rs_b200 as tb
    ins, d_out, d_w = make(1, 2, 90, 64, torch.float32, seed=7)
    got = run(ins, d_out, d_w)[2:]
    gen = torch.Generator().manual_seed(1)
    loss = lambda a: sum((x.double().cpu() * y.double()).sum().item() for x, y in zip(run(a), (d_out, d_w)))  # noqa: E731
    h = 2.0 ** -6
    for i, name in enumerate(("q", "k", "v", "g", "beta", "w")):
        d = torch.randn(ins[i].shape, generator=gen)
        up, down = list(ins), list(ins)
        up[i], down[i] = ins[i] + h * d, ins[i] - h * d
        slope, want = (got[i].double().cpu() * d.double()).sum().item(), (loss(up) - loss(down)) / (2 * h)
        size = (got[i].double().cpu().norm() * d.double().norm()).item()
        assert abs(slope - want) <= (2 ** -10 if name == "g" else 2 ** -11) * size, (name, slope, want, size)


def test_two_runs_are_the_same():
    ins, d_out, d_w = make(3, 4, 300, 64, torch.bfloat16, seed=8)
    a, b = run(ins, d_out, d_w), run(ins, d_out, d_w)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_state_that_is_never_handed_on_ends_the_launch():
    """The first block's range is taken by nobody: the block of the next one gives up its wait, reports it, and everything ends."""
    import ttt_rs_b200 as tb
    from ttt_rs_b200 import _lib
    lib = _lib.load()
    B, H = 50, 10
    # 500 streams of 10 chunks on 444 (backward: 296) blocks: the first one's 11 (16) steps end within a stream, which the second finishes
    ins, d_out, d_w = make(B, H, 640, 64, torch.bfloat16, seed=12)
    want = run(ins, d_out, d_w)
    tb.check_status()
    try:
        lib.ttt_b200_debug_handoff(2000, 1)
        with torch.no_grad():
            tb.fused_gated_linear(*[t.cuda() for t in ins])
        with pytest.raises(tb.TttError) as e:
            tb.check_status()
        assert e.value.code == _lib.TTT_ERR_TIMEOUT
        dev = [t.cuda().requires_grad_() for t in ins]
        lib.ttt_b200_debug_handoff(0, 0)
        out, _ = tb.fused_gated_linear(*dev)
        lib.ttt_b200_debug_handoff(2000, 1)
        torch.autograd.grad(out, dev, d_out.cuda())
        with pytest.raises(tb.TttError):
            tb.check_status()
    finally:
        lib.ttt_b200_debug_handoff(0, 0)
    assert all(torch.equal(x, y) for x, y in zip(run(ins, d_out, d_w), want))
    tb.check_status()


def test_captured_with_its_backward_and_replayed():
    """Forward and backward in one graph, replayed with other inputs in the captured buffers; few streams (segments) and many."""
    import ttt_rs_b200 as tb
    for B, H, T in ((1, 2, 700), (40, 12, 70)):
        ins, d_out, _ = make(B, H, T, 64, torch.bfloat16, seed=13)
        other, _, _ = make(B, H, T, 64, torch.bfloat16, seed=14)
        want = run(other, d_out)
        dev = [t.cuda() for t in ins]
        u = d_out.cuda()

        def step():
            leaves = [t.detach().requires_grad_() for t in dev]
            out, w = tb.fused_gated_linear(*leaves)
            return [out.detach(), w.detach(), *torch.autograd.grad(out, leaves, u)]
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for d, o in zip(dev, other):
            d.copy_(o)
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        tb.check_status()


def test_two_calls_at_once_on_two_streams():
    import ttt_rs_b200 as tb
    calls = []
    for seed, (B, H, T) in enumerate(((40, 12, 70), (40, 12, 70), (1, 3, 900), (1, 3, 900))):
        ins, _, _ = make(B, H, T, 64, torch.bfloat16, seed=20 + seed)
        calls.append(([t.cuda() for t in ins], run(ins)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    with torch.no_grad():
        for _ in range(3):
            got = []
            for (dev, _), s in zip(calls, streams):
                with torch.cuda.stream(s):
                    got.append(tb.fused_gated_linear(*dev))
    torch.cuda.synchronize()
    for (_, want), g in zip(calls, got):
        assert all(torch.equal(x, y) for x, y in zip(g, want))
    tb.check_status()


def test_refusals():
    import ttt_rs_b200 as tb
    ins, _, _ = make(1, 2, 8, 64, torch.bfloat16)
    dev = [t.cuda() for t in ins]

    def refused(code, **change):
        names = ("q", "k", "v", "g", "beta", "w")
        args = [change.get(n, t) for n, t in zip(names, dev)]
        with pytest.raises(tb.TttError) as e:
            tb.fused_gated_linear(*args)
        assert e.value.code == code

    from ttt_rs_b200 import _lib as L
    refused(L.TTT_ERR_SHAPE, k=dev[1][:, :1])
    refused(L.TTT_ERR_SHAPE, k=dev[1].float())
    refused(L.TTT_ERR_SHAPE, g=dev[3].bfloat16())
    refused(L.TTT_ERR_SHAPE, beta=dev[4][..., :4])
    refused(L.TTT_ERR_SHAPE, w=dev[5].bfloat16())
    refused(L.TTT_ERR_SHAPE, q=dev[0][0])
    refused(L.TTT_ERR_SHAPE, q=dev[0][:, :, :0], k=dev[1][:, :, :0], v=dev[2][:, :, :0], g=dev[3][..., :0], beta=None)
    refused(L.TTT_ERR_UNSUPPORTED, q=dev[0].half())
    refused(L.TTT_ERR_UNSUPPORTED, q=dev[0][..., :48], k=dev[1][..., :48], v=dev[2][..., :48])
    refused(L.TTT_ERR_CUDA, q=ins[0])


def test_saved_states_go_with_the_backward():
    """What the forward saves is freed by the backward, also while the results are kept."""
    import ttt_rs_b200 as tb
    ins, d_out, _ = make(4, 8, 1024, 64, torch.bfloat16)
    dev = [t.cuda().requires_grad_() for t in ins]
    torch.cuda.synchronize()
    out, w = tb.fused_gated_linear(*dev)
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(out, dev, d_out.cuda())
    held = torch.cuda.memory_allocated() - sum(t.numel() * t.element_size() for t in grads)
    assert held <= before - 4 * 8 * 16 * 64 * 64 * 4 + 65536
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(w, dev, torch.ones_like(w))


def test_gradients_of_gradients_are_refused():
    import ttt_rs_b200 as tb
    ins, _, _ = make(1, 2, 20, 64, torch.float32)
    dev = [t.cuda().requires_grad_() for t in ins]
    out, _ = tb.fused_gated_linear(*dev)
    want = torch.autograd.grad(out.sum(), dev, retain_graph=True)
    got = torch.autograd.grad(out.sum(), dev, create_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    with pytest.raises(RuntimeError, match="not differentiable"):
        sum(x.square().sum() for x in got).backward()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_finite_stays_in_its_stream_and_behind_its_chunk(bad):
    import ttt_rs_b200 as tb
    ins, _, _ = make(2, 2, 200, 64, torch.bfloat16, seed=6)
    want = run(ins)
    for x in ins[:3]:
        x[1, 0, 130] = bad
    got = run(ins)
    rest = torch.ones(2, 2, 200, dtype=torch.bool)
    rest[1, 0, 128:] = False
    assert torch.equal(got[0].cpu()[rest], want[0].cpu()[rest])
    assert not torch.isfinite(got[0][1, 0, 130:]).all(-1).any()
    others = torch.tensor([[True, True], [False, True]])
    assert torch.equal(got[1].cpu()[others], want[1].cpu()[others])
    tb.check_status()


def test_offsets_behind_32_bits():
    """9 sequences of 2^20 tokens and 4 heads as views of [B,T,H,F], 2.4e9 elements a tensor: the last tokens of the last stream against
    a call on those alone from the state before them."""
    import ttt_rs_b200 as tb
    B, H, T, F, last = 9, 4, 1 << 20, 64, 100
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(3, 1, T, H, F, generator=gen, device="cuda", dtype=torch.bfloat16)
    q, k, v = (t.expand(B, T, H, F).contiguous().transpose(1, 2) for t in x)
    decay = -0.3 * torch.rand(B, H, T, generator=gen, device="cuda")
    with torch.no_grad():
        out, _ = tb.fused_gated_linear(q, k, v, decay)
        cut = T - last
        _, state = tb.fused_gated_linear(q[-1:, :, :cut], k[-1:, :, :cut], v[-1:, :, :cut], decay[-1:, :, :cut])
        del q
        tail = [t[0].transpose(0, 1)[None, :, cut:].float() for t in x]
        want, _ = tb.fused_gated_linear(*tail, decay[-1:, :, cut:], None, state)
    tb.check_status()
    # bf16 results against float32 ones of the same inputs and (up to the order of their sums) the same state: three roundings
    mag, _ = tb.fused_gated_linear(*[t.abs() for t in tail], decay[-1:, :, cut:], None, state.abs())
    assert ((out[-1:, :, cut:].float() - want).abs() <= 3 * 2 ** -8 * mag + F32 * mag).all()


@pytest.mark.parametrize("reverse", [False, True])
def test_a_long_memory_keeps_its_digits(reverse):
    """128 chunks through a decay close to one, of as many streams as run without segments: the state (reverse: its gradient) as a
    whole.  It is rounded once per chunk, to nearest: at most 2^-24 of the largest state on the way each, 128 * 2^-24 = 2^-17 in all, the
    last of the states being the largest; a chunk's own part, of truncated sums of 12 products, 12 * 2^-23 of it, less than 2^-19.
    Together below 2^-16.  (Sums truncated onto the state itself lose 12 * 2^-24 of it per chunk on average, 2^-14 or half of that
    over a growing state.)"""
    import ttt_rs_b200 as tb
    B, H, T = 4, 37, 128 * 64
    gen = torch.Generator(device="cuda").manual_seed(8)
    q, k, v, u = torch.randn(4, B, H, T, 64, generator=gen, device="cuda").bfloat16()
    decay = torch.full((B, H, T), -2.0 ** -17, device="cuda")
    sums = torch.cumsum(decay.double(), -1)
    if reverse:
        w = torch.zeros(B, H, 64, 64, device="cuda").requires_grad_()
        out, _ = tb.fused_gated_linear(q, k, v, decay, None, w)
        (got,) = torch.autograd.grad(out, w, u)
        want = (q.double() * torch.exp(sums)[..., None]).transpose(2, 3) @ u.double()
    else:
        with torch.no_grad():
            _, got = tb.fused_gated_linear(q, k, v, decay)
        want = (k.double() * torch.exp(sums[..., -1:] - sums)[..., None]).transpose(2, 3) @ v.double()
    assert (got.double() - want).norm() <= 2 ** -16 * want.norm()
