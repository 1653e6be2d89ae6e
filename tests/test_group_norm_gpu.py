"""Group norm with channels last against its oracle: groups of every width, tokens and sequences, gates and activations."""

import pytest
import torch

import ttt_rs_b200 as tb
from mixer_checks import ELEMENT, SUM, close, grads, leaves
from oracle import mixer_oracle as O

pytestmark = pytest.mark.gpu

# B, T, groups, channels per group
TOKEN = [(2, 19, 3, 64), (1, 1, 1, 8), (8, 1, 24, 64), (2, 5, 7, 10), (3, 4, 5, 1), (2, 3, 2, 33), (1, 9, 1, 520), (2, 3, 1, 2047), (1, 2, 2, 4096),
         (2, 6, 40, 24), (3, 300, 4, 16)]
SEQUENCE = [(2, 19, 3, 64), (1, 1, 1, 8), (3, 40, 32, 10), (2, 5, 7, 3), (2, 3, 1, 2050), (1, 700, 2, 16), (2, 33, 1, 4096), (1, 2, 1, 9001)]


def make(B, T, G, c, dtype, affine=True, gate=True, at=0.5):
    g = torch.Generator().manual_seed(B * T + c)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    C = G * c
    return [(r(B, T, C) + at).to(dtype), (1 + 0.2 * r(C)).to(dtype) if affine else None, (0.3 * r(C)).to(dtype) if affine else None,
            r(B, T, C).to(dtype) if gate else None], r(B, T, C).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("how", [dict(activation="silu"), dict(activation="silu", gate=False), dict(activation="gelu", gate=False, affine=False),
                                 dict(activation=None, gate=False), dict(activation="gelu")], ids=lambda h: "-".join(map(str, h.values())))
@pytest.mark.parametrize("over,case", [("token", c) for c in TOKEN] + [("sequence", c) for c in SEQUENCE], ids=str)
def test_results_and_gradients(over, case, how, dtype):
    B, T, G, c = case
    ins, up = make(*case, dtype, how.get("affine", True), how.get("gate", True))
    dev, ref = leaves(ins)
    call = lambda f, t: f(t[0], G, t[1], t[2], gate=t[3], activation=how["activation"], eps=1e-3, over=over)  # noqa: E731
    y, want = call(tb.group_norm, dev), call(O.group_norm, ref)
    close(y, want, "y")
    with torch.no_grad():
        assert torch.equal(call(tb.group_norm, dev), y)
    # gradients: the difference from two means, each a sum of the group
    got, exp = grads(y, dev, up.cuda()), grads(want, ref, up.double())
    names = [n for n, t in zip(("x", "weight", "bias", "gate"), ins) if t is not None]
    if c == 1 and over == "token":  # n is 0 throughout: nothing but roundings of zero in x's and the weight's gradients
        got, exp, names = zip(*[t for t in zip(got, exp, names) if t[2] not in ("x", "weight")] or [((), (), ())]) if len(names) > 1 else ((), (), ())
    for a, b, n in zip(got, exp, names):
        close(a, b, n, SUM if n in ("weight", "bias") else 4 * ELEMENT)


@pytest.mark.parametrize("over", ["token", "sequence"])
def test_views_of_a_projection(over):
    ins, up = make(3, 12, 4, 16, torch.bfloat16)
    wide = torch.randn(3, 12, 200, device="cuda").bfloat16()
    wide[..., 8:72], wide[..., 72:136] = ins[0].cuda(), ins[3].cuda()
    w, b = ins[1].cuda(), ins[2].cuda()
    want = tb.group_norm(ins[0].cuda(), 4, w, b, gate=ins[3].cuda(), activation="silu", over=over)
    assert torch.equal(tb.group_norm(wide[..., 8:72], 4, w, b, gate=wide[..., 72:136], activation="silu", over=over), want)
    odd = torch.randn(3, 12, 131, device="cuda").bfloat16()
    odd[..., 3:67] = ins[0].cuda()
    got = tb.group_norm(odd[..., 3:67], 4, w, b, gate=ins[3].cuda(), activation="silu", over=over)
    close(got, want.double(), "odd address", arithmetic=2.0 ** -8)  # (another order of the sums may round otherwise, once)
    turned = ins[0].cuda().transpose(0, 1).contiguous().transpose(0, 1)  # [B,T,C] of [T,B,C]
    assert torch.equal(tb.group_norm(turned, 4, w, b, gate=ins[3].cuda(), activation="silu", over=over), want)
    x = ins[0].cuda().requires_grad_()
    g1 = torch.autograd.grad(tb.group_norm(x, 4, w, b, over=over), x, up.cuda())[0]
    g2 = torch.autograd.grad(tb.group_norm(x, 4, w, b, over=over), x, up.cuda().transpose(0, 1).contiguous().transpose(0, 1))[0]
    assert torch.equal(g1, g2)


@pytest.mark.parametrize("over", ["token", "sequence"])
def test_variances_do_not_cancel(over):
    """A mean of 1000 standard deviations: sums of squares would leave nothing of the variance in float32."""
    ins, _ = make(2, 64, 2, 256, torch.float32, gate=False, at=1000.0)
    dev, ref = leaves(ins)
    y = tb.group_norm(*dev[:1], 2, *dev[1:3], over=over)
    # inputs near 1000 are given exactly; a mean that is off by 2^-24 of 1000 (its own rounding) shifts a result by 6e-5
    close(y, O.group_norm(ref[0], 2, *ref[1:3], over=over), "y", arithmetic=2.0 ** -12)


def test_what_is_not_finite_stays_in_its_group():
    x = torch.randn(2, 6, 64, device="cuda")
    x[1, 3, 20] = float("nan")
    x[0, 2, 50] = float("inf")
    y = tb.group_norm(x, 4)
    bad = torch.zeros(2, 6, 4, dtype=torch.bool, device="cuda")
    bad[1, 3, 1] = bad[0, 2, 3] = True
    assert torch.equal(y.unflatten(-1, (4, 16)).isnan().any(-1), bad)
    y = tb.group_norm(x, 4, over="sequence")
    assert torch.equal(y.unflatten(-1, (4, 16)).isnan().any(-1).any(1), bad.any(1))


def test_constant_groups():
    x = torch.full((2, 3, 32), 3.0, device="cuda", requires_grad=True)
    b = torch.randn(32, device="cuda")
    y = tb.group_norm(x, 2, None, b)
    assert torch.equal(y, b.expand(2, 3, 32))
    assert torch.isfinite(torch.autograd.grad(y.sum(), x)[0]).all()


def test_graph_capture_and_order():
    """A captured training step gives the eager one's results, run after run."""
    ins, up = make(4, 50, 4, 32, torch.bfloat16)
    dev = [t.cuda().requires_grad_() for t in ins]
    up = up.cuda()
    for over in ("token", "sequence"):
        step = lambda: torch.autograd.grad(tb.group_norm(dev[0], 4, dev[1], dev[2], gate=dev[3], activation="silu", over=over), dev, up)  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [t.clone() for t in step()]
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        for _ in range(2):
            for t in got:
                t.zero_()
            g.replay()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    x = torch.randn(2, 3, 32, device="cuda")
    w = torch.ones(32, device="cuda")
    for f in (lambda: tb.group_norm(x, 5), lambda: tb.group_norm(x, 0), lambda: tb.group_norm(x, 4, w[:16]), lambda: tb.group_norm(x, 4, w.bfloat16()),
              lambda: tb.group_norm(x, 4, gate=x[:1]), lambda: tb.group_norm(x, 4, activation="relu"), lambda: tb.group_norm(x, 4, over="batch"),
              lambda: tb.group_norm(x[0], 4), lambda: tb.group_norm(x[:, :0], 4), lambda: tb.group_norm(x.half(), 4),
              lambda: tb.group_norm(torch.zeros(1, 1, 5000, device="cuda"), 1), lambda: tb.group_norm(x, 4, eps=-1.0)):
        with pytest.raises(tb.TttError):
            f()
    xg = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(tb.group_norm(xg, 4).square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
