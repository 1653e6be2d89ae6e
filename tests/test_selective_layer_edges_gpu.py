"""Edges of the selective layer's operators: an epsilon of zero, rates of -inf, steps of zero, GELU of large numbers."""

import pytest
import torch

import ttt_rs_b200 as tb
from mixer_checks import ELEMENT, SUM, close, grads, leaves
from oracle import mixer_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("over", ["token", "sequence"])
@pytest.mark.parametrize("case", [(3, 29, 4, 16), (1, 5, 2, 33), (2, 7, 3, 6), (1, 3, 2, 520)], ids=str)
def test_an_epsilon_of_zero(case, over, gated, dtype):
    """Blocks whose last rows hold no token: 1 / sqrt(0 + 0) of nothing must not reach the sums for weight and bias."""
    B, T, G, c = case
    g = torch.Generator().manual_seed(T + c)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    C = G * c
    ins = [r(B, T, C).to(dtype), (1 + 0.2 * r(C)).to(dtype), (0.3 * r(C)).to(dtype), r(B, T, C).to(dtype) if gated else None]
    up = r(B, T, C).to(dtype)
    dev, ref = leaves(ins)
    call = lambda f, t: f(t[0], G, t[1], t[2], gate=t[3], activation="silu", eps=0.0, over=over)  # noqa: E731
    y, want = call(tb.group_norm, dev), call(O.group_norm, ref)
    close(y, want, "y")
    for a, b, n in zip(grads(y, dev, up.cuda()), grads(want, ref, up.double()), ("x", "weight", "bias", "gate")):
        close(a, b, n, SUM if n in ("weight", "bias") else 4 * ELEMENT)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("N", [16, 10])
@pytest.mark.parametrize("T", [1, 16, 21, 700])
def test_a_step_of_zero_keeps_a_state_at_any_rate(T, N, dtype):
    """A rate of -inf keeps nothing over a step above zero and everything over a step of zero, as its limit, the lowest rate, does:
    in single tokens, in short calls and in long ones."""
    g = torch.Generator().manual_seed(T + N)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    B, C = 2, 24
    x, dt = (0.5 * r(B, T, C)).to(dtype), (0.5 * r(B, T, C)).to(dtype)
    dt[0, :, :8] = -200.0  # (a step of zero in float32)
    dt[1, T // 2:, 4:] = float("-inf")
    A = -torch.exp(0.7 * r(C, N))
    A[:, 3] = float("-inf")
    Bm, Cm, bias, state = r(B, T, 1, N).to(dtype), r(B, T, 1, N).to(dtype), 0.5 * r(C) - 1.0, r(B, C, N)
    lowest = A.double().clamp(min=torch.finfo(torch.float32).min)
    want = O.selective_scan(x.double(), dt.double(), lowest, Bm.double(), Cm.double(), None, None, bias.double(), state.double())
    t = [v.cuda() for v in (x, dt, A, Bm, Cm)]
    for recorded in (False, True):  # (recorded for gradients, few tokens are scanned as many are)
        t[0].requires_grad_(recorded)
        y, s = tb.selective_scan(*t, dt_bias=bias.cuda(), state=state.cuda())
        close(y, want[0], "y", 2 * ELEMENT)
        close(s, want[1], "state", 2 * ELEMENT)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("N", [16, 10])
@pytest.mark.parametrize("T", [1, 21, 700])
def test_gradients_at_steps_of_zero_and_rates_of_minus_infinity(T, N, dtype):
    """The lowest rate times a state's gradient may be beyond float32, the softplus's slope there is zero: no gradient for the step."""
    g = torch.Generator().manual_seed(T + N)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    B, C = 2, 24
    x, dt = (0.5 * r(B, T, C)).to(dtype), (0.5 * r(B, T, C)).to(dtype)
    dt[0, :, :8] = -200.0
    dt[1, T // 2:, 4:] = float("-inf")
    A = -torch.exp(0.7 * r(C, N))
    A[:, 3] = A[:, 7] = torch.finfo(torch.float32).min
    ins = [x, dt, A, r(B, T, 1, N).to(dtype), r(B, T, 1, N).to(dtype), None, None, 0.5 * r(C) - 1.0, 8 * r(B, C, N)]
    dev, ref = leaves(ins)
    dev[2] = torch.where(ins[2] == ins[2].min(), float("-inf"), ins[2]).cuda().requires_grad_()
    call = lambda f, t: f(*t[:5], dt_bias=t[7], state=t[8])  # noqa: E731
    outs, want = call(tb.selective_scan, dev), call(O.selective_scan, ref)
    up = [r(*w.shape).to(o.dtype) for o, w in zip(outs, want)]
    got, exp = grads(outs, dev, [8 * u.cuda() for u in up]), grads(want, ref, [8 * u.double() for u in up])
    for a, b, n in zip(got, exp, ("x", "dt", "A", "B", "C", "dt_bias", "state")):
        close(a, b, n, SUM)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [1e10, 1e20, 3e38])
@pytest.mark.parametrize("over", ["token", "sequence"])
def test_gelu_of_large_numbers(over, size, dtype):
    """GELU's slope is 1 and 0 far from zero, also where the cube, or the square, of its argument is beyond float32."""
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    B, T, G, C = 2, 9, 2, 32
    ends = torch.where(torch.arange(C) % 3 == 0, size, torch.where(torch.arange(C) % 3 == 1, -size, 0.5))
    x, up = r(B, T, C).to(dtype), r(B, T, C).to(dtype)
    # as the gate: its gradient
    dev, ref = leaves([x, None, None, ends.expand(B, T, C).contiguous().to(dtype)])
    call = lambda f, t: f(t[0], G, t[1], t[2], gate=t[3], activation="gelu", eps=1e-3, over=over)  # noqa: E731
    (got,) = torch.autograd.grad(call(tb.group_norm, dev), dev[3], up.cuda())
    (exp,) = torch.autograd.grad(call(O.group_norm, ref), ref[3], up.double())
    close(got, exp, "gate")
    # as the normed and shifted input: the others' gradients
    dev, ref = leaves([x, (1 + 0.2 * r(C)).to(dtype), ends.to(dtype), None])
    got, exp = grads(call(tb.group_norm, dev), dev, up.cuda()), grads(call(O.group_norm, ref), ref, up.double())
    for a, b, n in zip(got, exp, ("x", "weight", "bias")):
        close(a, b, n, SUM if n != "x" else 4 * ELEMENT)
