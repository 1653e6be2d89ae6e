"""Selective state space scan against its oracle: states, groups, types, odd sizes, strides, carried states, starts, segments,
gradients."""

import pytest
import torch

import ttt_rs_b200 as tb
from mixer_checks import ELEMENT, SUM, close, grads, leaves
from oracle import mixer_oracle as O

pytestmark = pytest.mark.gpu
NAMES = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state")


def make(B, T, C, N, G=1, dtype=torch.float32, seed=0, skip=True, gate=True, bias=True, state=True, starts=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    marks = None
    if starts:
        marks = torch.rand(B, T, generator=g) < 0.1
        if T > 2:  # a row without a start, and one that begins with one
            marks[0, :] = False
            marks[-1, 0] = True
    return [(0.5 * r(B, T, C)).to(dtype), (0.5 * r(B, T, C)).to(dtype), -torch.exp(0.7 * r(C, N)), r(B, T, G, N).to(dtype), r(B, T, G, N).to(dtype),
            r(C) if skip else None, r(B, T, C).to(dtype) if gate else None, 0.5 * r(C) - 1.0 if bias else None,
            r(B, C, N) if state else None], marks


def scan(f, t, marks, **kw):
    return f(t[0], t[1], t[2], t[3], t[4], t[5], z=t[6], dt_bias=t[7], state=t[8], starts=marks, **kw)


CASES = [
    # B, T, C, N, G, what is there
    (2, 37, 64, 16, 1, {}), (1, 16, 8, 16, 1, {}), (1, 17, 136, 16, 1, dict(gate=False)), (2, 33, 40, 16, 2, dict(starts=False)),
    (2, 20, 7, 16, 1, {}), (1, 50, 6, 10, 3, {}), (2, 19, 130, 8, 1, dict(skip=False, bias=False)), (1, 40, 140, 4, 1, {}), (1, 21, 33, 3, 1, {}),
    (2, 35, 48, 32, 1, {}), (1, 18, 20, 64, 2, {}), (1, 31, 9, 33, 1, dict(state=False)), (1, 5, 24, 1, 1, {}), (1, 1, 72, 16, 1, {}),
    (1, 700, 16, 16, 1, {}), (2, 1000, 24, 8, 2, dict(starts=False)),  # segments
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_results_and_gradients(case, dtype):
    B, T, C, N, G, what = case
    ins, marks = make(B, T, C, N, G, dtype, seed=T + C, **what)
    dev, ref = leaves(ins)
    on = None if marks is None else marks.cuda()
    outs, want = scan(tb.selective_scan, dev, on), scan(O.selective_scan, ref, marks)
    # a state is a sum of decayed terms: as many float32 operations as tokens that are not yet forgotten
    for o, w, n in zip(outs, want, ("y", "state")):
        close(o, w, n, 2 * ELEMENT)
    with torch.no_grad():
        plain = scan(tb.selective_scan, dev, on)  # (without gradients: a decode step of up to 16 tokens, which sums otherwise)
        for o, w, n in zip(plain, want, ("y", "state")):
            close(o, w, n, 2 * ELEMENT)
    g = torch.Generator().manual_seed(7)
    up = [torch.randn(w.shape, generator=g).to(o.dtype) for w, o in zip(want, outs)]
    names = [n for n, t in zip(NAMES, ins) if t is not None]
    got, exp = grads(outs, dev, [u.cuda() for u in up]), grads(want, ref, [u.double() for u in up])
    for a, b, n in zip(got, exp, names):
        close(a, b, n, SUM)


def test_one_result_alone_and_plain_steps():
    ins, marks = make(2, 40, 24, 16)
    ins[1], ins[7] = ins[1].abs(), ins[7].abs()  # softplus=False: steps as they are (negative ones grow beyond float32)
    for k in (0, 1):
        dev, ref = leaves(ins)
        outs = scan(tb.selective_scan, dev, marks.cuda(), softplus=False)
        want = scan(O.selective_scan, ref, marks, softplus=False)
        use = [0, 1, 2, 3, 8] if k == 1 else list(range(9))
        got = torch.autograd.grad(outs[k].sum(), [dev[i] for i in use])
        exp = torch.autograd.grad(want[k].sum(), [ref[i] for i in use])
        for a, b, i in zip(got, exp, use):
            close(a, b, NAMES[i], SUM)


def test_views_of_projections():
    ins, marks = make(2, 45, 32, 16, dtype=torch.bfloat16)
    want = scan(tb.selective_scan, [t.cuda() for t in ins], marks.cuda())
    wide = torch.randn(2, 45, 32 * 3 + 32 + 8, device="cuda").bfloat16()
    views = list(ins)
    for i, (n, at, w) in enumerate((("x", 0, 32), ("dt", 32, 32), ("z", 64, 32))):
        k = NAMES.index(n)
        wide[..., at:at + w] = ins[k].cuda()
        views[k] = wide[..., at:at + w]
    for n, at in (("B", 96), ("C", 112)):
        wide[..., at:at + 16] = ins[NAMES.index(n)][:, :, 0].cuda()
        views[NAMES.index(n)] = wide[..., at:at + 16]  # [B,T,N]: one group
    on = [t if t is None or t.is_cuda else t.cuda() for t in views]
    got = scan(tb.selective_scan, on, marks.cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.randn(2, 45, 101, device="cuda").bfloat16()  # rows off every vector's address
    odd[..., 3:35], odd[..., 35:67], odd[..., 67:83] = ins[0].cuda(), ins[6].cuda(), ins[3][:, :, 0].cuda()
    on[0], on[6], on[3] = odd[..., 3:35], odd[..., 35:67], odd[..., 67:83]
    got = scan(tb.selective_scan, on, marks.cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_token_by_token_is_the_sequence(dtype):
    ins, marks = make(3, 90, 48, 16, dtype=dtype)
    ref = [None if t is None else t.double() for t in ins]
    t = [v.cuda() for v in ins]
    marks_on = marks.cuda()
    want = scan(O.selective_scan, ref, marks)
    state, outs, at = t[8].clone(), [], 0
    for n in (1, 1, 16, 2, 17, 1, 30, 22):  # steps and short sequences, the state advanced where it lies
        part = [v[:, at:at + n] if v.dim() >= 3 and v.shape[1] == 90 else v for v in t[:8]] + [state]
        y, state2 = scan(tb.selective_scan, part, marks_on[:, at:at + n], state_out=state)
        assert state2 is state
        outs.append(y)
        at += n
    assert at == 90
    close(torch.cat(outs, 1), want[0], "y", 2 * ELEMENT)
    close(state, want[1], "state", 2 * ELEMENT)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,C,N,G", [(64, 640, 16, 1), (64, 640, 10, 5), (40, 256, 64, 1), (160, 1000, 3, 1), (64, 1300, 8, 2), (33, 700, 32, 7)])
def test_steps_of_many_sequences(B, C, N, G, dtype):
    """Steps whose threads would not all be resident hold more states each."""
    ins, marks = make(B, 2, C, N, G, dtype, starts=True)
    got = scan(tb.selective_scan, [t.cuda() for t in ins], marks.cuda())
    want = scan(O.selective_scan, [t.double() for t in ins], marks)
    close(got[0], want[0], "y", 2 * ELEMENT)
    close(got[1], want[1], "state", 2 * ELEMENT)


def test_a_state_in_place_over_segments():
    ins, _ = make(1, 3000, 16, 16, dtype=torch.bfloat16, starts=False)
    t = [v.cuda() for v in ins]
    want = scan(tb.selective_scan, t, None)
    state = t[8].clone()
    got = scan(tb.selective_scan, t[:8] + [state], None, state_out=state)
    assert torch.equal(got[0], want[0]) and torch.equal(state, want[1])


@pytest.mark.parametrize("T", [12, 40, 2000])
def test_a_start_hides_what_is_not_finite(T):
    ins, _ = make(2, T, 24, 16)
    marks = torch.zeros(2, T, dtype=torch.bool)
    cut = T // 2 + 3
    marks[:, cut] = True
    ins[0][:, cut - 2:cut] = float("nan")
    dev = [t.cuda().requires_grad_() for t in ins]
    y, s = scan(tb.selective_scan, dev, marks.cuda())
    assert torch.isfinite(y[:, cut:]).all() and torch.isfinite(s).all() and torch.isfinite(y[:, :cut - 2]).all()
    (gs,) = torch.autograd.grad(y[:, cut:].sum() + s.sum(), dev[8])
    assert not gs.any()  # nothing behind the start depends on the state
    with torch.no_grad():
        y, s = scan(tb.selective_scan, dev, marks.cuda())
        assert torch.isfinite(y[:, cut:]).all() and torch.isfinite(s).all() and torch.isfinite(y[:, :cut - 2]).all()


def test_long_memory_keeps_its_precision():
    """Decays of 2^-12 per token over 8192 tokens: thousands of products of numbers next to one.  Their float32 roundings, and the
    approximate exponential's, must not all lean the same way: 4096 tokens' memory times 2^-25 each way at random is 2^-19 of the
    state; 2^-16 leaves room for a bias of 2^-28 per token."""
    T = 8192
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, T, 8, generator=g) + 1.0
    dt = torch.full((1, T, 8), 2.0 ** -6)
    A = torch.full((8, 4), -(2.0 ** -6))
    A[:, 1] *= 2
    Bm, Cm = torch.ones(1, T, 1, 4), torch.ones(1, T, 1, 4)
    args = [x, dt, A, Bm, Cm, None, None, None, None]
    y, s = scan(tb.selective_scan, [None if t is None else t.cuda() for t in args], None, softplus=False)
    want = scan(O.selective_scan, [None if t is None else t.double() for t in args], None, softplus=False)
    close(y, want[0], "y", 2.0 ** -16)
    close(s, want[1], "state", 2.0 ** -16)


def test_extreme_steps():
    """Steps that forget everything, and steps of zero."""
    ins, _ = make(1, 40, 8, 16, starts=False, gate=False)
    ins[1][:, 10] = 300.0
    ins[1][:, 20] = -200.0
    ins[1][:, 30] = float("-inf")
    dev, ref = leaves(ins)
    outs, want = scan(tb.selective_scan, dev, None), scan(O.selective_scan, ref, None)
    close(outs[0], want[0], "y", 2 * ELEMENT)
    close(outs[1], want[1], "state", 2 * ELEMENT)


def test_rates_that_keep_nothing():
    """A rate of -inf keeps nothing of a state, in sequences of any length: 0 = exp(-inf) for every step above zero."""
    ins, _ = make(1, 21, 8, 16, starts=False)
    ins[2][:, 3] = float("-inf")
    t = [v.cuda() for v in ins]
    y, s = scan(tb.selective_scan, t, None)
    want = scan(O.selective_scan, [v.double() for v in ins], None)
    close(y, want[0], "y", 2 * ELEMENT)
    close(s, want[1], "state", 2 * ELEMENT)


def test_graph_capture_of_steps_and_training():
    ins, _ = make(4, 1, 64, 16, dtype=torch.bfloat16, starts=False)
    t = [v.cuda() for v in ins]
    state = t[8].clone()
    scan(tb.selective_scan, t, None)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, _ = scan(tb.selective_scan, t[:8] + [state], None, state_out=state)
    want = t[8]
    for _ in range(3):
        g.replay()
        y2, want = scan(tb.selective_scan, t[:8] + [want], None)
        assert torch.equal(y, y2) and torch.equal(state, want)

    ins, marks = make(1, 600, 32, 16, dtype=torch.bfloat16)
    dev = [v.cuda().requires_grad_() for v in ins]
    marks = marks.cuda()
    step = lambda: torch.autograd.grad(scan(tb.selective_scan, dev, marks)[0].float().sum(), dev[:8])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [v.clone() for v in step()]
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(2):
        for v in got:
            v.zero_()
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    """Calls on two streams have workspaces of their own."""
    ins, marks = make(1, 5000, 64, 16, dtype=torch.bfloat16)
    t, marks = [v.cuda() for v in ins], marks.cuda()
    want = scan(tb.selective_scan, t, marks)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(scan(tb.selective_scan, t, marks))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in got)


def test_offsets_behind_32_bits():
    B, T, C = 1, 40000, 65536
    x = torch.zeros(B, T, C, device="cuda", dtype=torch.bfloat16)
    x[0, -2:] = 1.0
    dt = torch.zeros(1, 1, C, device="cuda", dtype=torch.bfloat16).expand(B, T, C)
    A = torch.full((C, 4), -1.0, device="cuda")
    b = torch.ones(B, T, 4, device="cuda", dtype=torch.bfloat16)
    y, s = tb.selective_scan(x, dt, A, b, b)
    d = torch.log(torch.tensor(2.0, dtype=torch.float64))
    h = d * torch.exp(-d) + d
    close(s, h.expand(1, C, 4), "state")
    close(y[0, -2:], torch.stack([4 * d, 4 * h])[:, None].expand(2, C), "y")
    assert not y[0, :-2].any()


def test_refusals():
    ins, marks = make(2, 9, 16, 8)
    t, marks = [v.cuda() for v in ins], marks.cuda()

    def call(*, kw=None, **new):
        v = list(t)
        for n, e in new.items():
            v[NAMES.index(n)] = e
        return lambda: scan(tb.selective_scan, v, marks, **(kw or {}))
    x = t[0]
    bad = [call(dt=t[1][:, :3]), call(dt=t[1].bfloat16()), call(A=t[2].bfloat16()), call(A=t[2][:, :4]), call(B=t[3][:, :, :, :4]), call(B=t[3].expand(2, 9, 3, 8)),
           call(C=t[4].bfloat16()), call(D=t[5][:3]), call(z=t[6][:1]), call(dt_bias=t[7].bfloat16()), call(state=t[8][:, :, :4]), call(x=x[0]),
           call(x=x.half()), call(state=t[8].bfloat16()), call(kw=dict(state_out=t[8][:1])), call(kw=dict(state_out=t[8].bfloat16())),
           call(B=torch.zeros(2, 9, 1, 65, device="cuda"), C=torch.zeros(2, 9, 1, 65, device="cuda"), A=torch.zeros(16, 65, device="cuda"), state=None)]
    for i, f in enumerate(bad):
        with pytest.raises(tb.TttError):
            f()
            print("not refused:", i)
    with pytest.raises(tb.TttError):
        scan(tb.selective_scan, t, marks[:, :3])
    # a result over another tensor of the call
    pool = torch.zeros(2 * 16 * 8 + 16, device="cuda")
    with pytest.raises(tb.TttError):
        scan(tb.selective_scan, t[:8] + [pool[:256].view(2, 16, 8)], marks, state_out=pool[16:].view(2, 16, 8))
    with pytest.raises(tb.TttError):  # results that are given are not recorded
        scan(tb.selective_scan, [x.clone().requires_grad_()] + t[1:], marks, state_out=t[8])
    xg = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(scan(tb.selective_scan, [xg] + t[1:], marks)[0].square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):  # once differentiable
        gx.sum().backward()
