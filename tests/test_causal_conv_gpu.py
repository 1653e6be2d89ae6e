"""Causal convolution against its oracle: taps, types, odd sizes, strides, carried states, starts, gradients."""

import pytest
import torch

import ttt_rs_b200 as tb
from mixer_checks import ELEMENT, SUM, close, grads, leaves
from oracle import mixer_oracle as O

pytestmark = pytest.mark.gpu


def make(B, T, C, K, dtype, seed=0, bias=True, state=True, starts=True, columns=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    x = r(B, T, C + 24)[..., 8:8 + C] if columns else r(B, T, C)
    marks = torch.rand(B, T, generator=g) < 0.2 if starts else None
    if starts and T > 2:
        marks[0, :] = False  # a row without a start, and one that begins with one
        marks[-1, 0] = True
    return [x, r(C, K), r(C) if bias else None, r(B, K - 1, C) if state else None], marks


CASES = [
    # B, T, C, K, what is there
    (2, 37, 64, 4, {}), (1, 1, 16, 4, {}), (3, 2, 24, 4, {}), (2, 3, 8, 4, {}), (1, 33, 1, 2, {}), (2, 17, 7, 3, {}),
    (2, 64, 40, 2, dict(starts=False)), (1, 100, 264, 4, dict(state=False)), (2, 31, 12, 3, dict(bias=False, state=False, starts=False)),
    (2, 45, 32, 4, dict(columns=True)), (5, 16, 2050, 4, {}),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_results_and_gradients(case, activation, dtype):
    B, T, C, K, what = case
    ins, marks = make(B, T, C, K, dtype, seed=T + C, **what)
    dev, ref = leaves(ins)
    if what.get("columns"):  # (leaves are made contiguous: a column block is a view of one)
        wide = torch.zeros(B, T, C + 24, device="cuda", dtype=dtype)
        wide[..., 8:8 + C] = ins[0].cuda()
        dev[0] = wide.requires_grad_()
        x = dev[0][..., 8:8 + C]
    else:
        x = dev[0]
    on = None if marks is None else marks.cuda()
    outs = tb.causal_conv(x, dev[1], dev[2], dev[3], activation=activation, starts=on)
    want = O.causal_conv(*ref, activation=activation, starts=marks)
    g = torch.Generator().manual_seed(7)
    up = [torch.randn(w.shape, generator=g).to(dtype) for w in want]
    close(outs[0], want[0], "y")
    assert torch.equal(outs[1].cpu().double(), want[1].detach())  # (copies)
    with torch.no_grad():
        plain = tb.causal_conv(x, dev[1], dev[2], dev[3], activation=activation, starts=on)
        assert torch.equal(plain[0], outs[0]) and torch.equal(plain[1], outs[1])
    got = grads(outs, dev, [u.cuda() for u in up])
    ref_grads = grads(want, ref, [u.double() for u in up])
    for i, (a, b) in enumerate(zip(got, ref_grads)):
        if i == 0 and what.get("columns"):
            assert not a[..., :8].any() and not a[..., 8 + C:].any()
            a = a[..., 8:8 + C]
        close(a, b, f"gradient {i}", SUM if i in (1, 2) else ELEMENT)


def test_one_result_alone_and_frozen_inputs():
    ins, marks = make(2, 20, 16, 4, torch.float32)
    for k in (0, 1):
        dev, ref = leaves(ins)
        outs, want = tb.causal_conv(*dev, starts=marks.cuda()), O.causal_conv(*ref, starts=marks)
        got = torch.autograd.grad(outs[k].sum(), [dev[0], dev[3]])
        exp = torch.autograd.grad(want[k].sum(), [ref[0], ref[3]], allow_unused=True)  # (the new state has nothing of the given one)
        for a, b, t in zip(got, exp, (ref[0], ref[3])):
            close(a, torch.zeros_like(t) if b is None else b, f"result {k}")
    x = ins[0].cuda().requires_grad_()
    (gx,) = torch.autograd.grad(tb.causal_conv(x, *[t.cuda() for t in ins[1:]])[0].sum(), x)
    assert gx.shape == x.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_token_by_token_is_the_sequence(dtype):
    (x, w, b, s), marks = make(3, 41, 48, 4, dtype)
    x, w, b, s, marks = (t.cuda() for t in (x, w, b, s, marks))
    whole, end = tb.causal_conv(x, w, b, s, activation="silu", starts=marks)
    state, outs, at = s.clone(), [], 0
    for n in (1, 1, 2, 3, 1, 20, 13):  # the state advanced where it lies
        y, state2 = tb.causal_conv(x[:, at:at + n], w, b, state, activation="silu", starts=marks[:, at:at + n], state_out=state)
        assert state2 is state
        outs.append(y)
        at += n
    assert at == 41 and torch.equal(torch.cat(outs, 1), whole) and torch.equal(state, end)


def test_a_start_hides_what_is_not_finite():
    (x, w, b, s), _ = make(2, 30, 16, 4, torch.float32)
    marks = torch.zeros(2, 30, dtype=torch.bool)
    marks[:, 10] = True
    x[:, 7:10] = float("nan")
    y, _ = tb.causal_conv(x.cuda(), w.cuda(), b.cuda(), s.cuda(), activation="silu", starts=marks.cuda())
    assert torch.isfinite(y[:, 10:]).all() and torch.isfinite(y[:, :7]).all() and y[:, 7:10].isnan().all()


def test_offsets_behind_32_bits():
    """Rows of a tensor of more than 2^31 elements, the last ones read and written."""
    B, T, C = 1, 70000, 32768
    x = torch.zeros(B, T, C, device="cuda", dtype=torch.bfloat16)
    x[0, -4:] = torch.randn(4, C, device="cuda")
    w = torch.randn(C, 4, device="cuda", dtype=torch.bfloat16)
    y, s = tb.causal_conv(x, w)
    want = (x[0, -4:].float() * w.t().float()).sum(0)
    assert torch.equal(s[0], x[0, -3:])
    close(y[0, -1], want, "last token")


def test_graph_capture_and_streams():
    (x, w, b, s), _ = make(4, 1, 64, 4, torch.bfloat16, starts=False)
    x, w, b, s = (t.cuda() for t in (x, w, b, s))
    state = s.clone()
    tb.causal_conv(x, w, b, state, activation="silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        y, _ = tb.causal_conv(x, w, b, state, activation="silu", state_out=state)
    want = s.clone()
    for _ in range(3):
        g.replay()
        y2, want = tb.causal_conv(x, w, b, want, activation="silu")
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and torch.equal(state, want)


def test_refusals():
    (x, w, b, s), marks = make(2, 9, 16, 4, torch.float32)
    x, w, b, s, marks = (t.cuda() for t in (x, w, b, s, marks))
    bad = [lambda: tb.causal_conv(x, w[:, :1].contiguous()), lambda: tb.causal_conv(x, torch.cat([w, w], 1)), lambda: tb.causal_conv(x, w[:8]),
           lambda: tb.causal_conv(x, w.bfloat16()), lambda: tb.causal_conv(x, w, b[:8]), lambda: tb.causal_conv(x, w, b, s[:, :2]),
           lambda: tb.causal_conv(x, w, activation="gelu"), lambda: tb.causal_conv(x, w, starts=marks[:, :3]),
           lambda: tb.causal_conv(x, w, starts=marks.float()), lambda: tb.causal_conv(x[0], w), lambda: tb.causal_conv(x[:, :0], w),
           lambda: tb.causal_conv(x.half(), w.half()), lambda: tb.causal_conv(x, w, state=s, state_out=x[:, :3]),
           lambda: tb.causal_conv(x, w, state=s, state_out=s.transpose(0, 1).contiguous().transpose(0, 1))]
    for f in bad:
        with pytest.raises(tb.TttError):
            f()
    with pytest.raises(tb.TttError):  # results that are given are not recorded
        tb.causal_conv(x.clone().requires_grad_(), w, state=s, state_out=s)
    with pytest.raises(RuntimeError):  # once differentiable
        xg = x.clone().requires_grad_()
        (gx,) = torch.autograd.grad(tb.causal_conv(xg, w)[0].square().sum(), xg, create_graph=True)
        gx.sum().backward()


def test_a_state_that_a_backward_needs_counts_as_overwritten():
    (x, w, b, s), _ = make(2, 9, 16, 4, torch.float32)
    wg, s = w.cuda().requires_grad_(), s.cuda()
    y, _ = tb.causal_conv(x.cuda(), wg, state=s)
    with torch.no_grad():
        tb.causal_conv(x.cuda(), wg, state=s, state_out=s)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
