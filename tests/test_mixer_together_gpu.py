"""The selective layer's operators in a run together: input projection, causal convolution, scan, gated group norm, output
projection, as a layer trains with them and as it generates."""

import pytest
import torch

import ttt_rs_b200 as tb
from mixer_checks import close
from oracle import mixer_oracle as O

pytestmark = pytest.mark.gpu

HIDDEN, WIDE, STATES, RANK, HEADS = 48, 96, 16, 8, 6


def weights(seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: torch.randn(*s, generator=g, dtype=torch.float64) * scale  # noqa: E731
    return dict(inp=r(2 * WIDE, HIDDEN, scale=HIDDEN ** -0.5), conv=r(WIDE, 4, scale=0.5), conv_bias=r(WIDE, scale=0.1),
                xp=r(RANK + 2 * STATES, WIDE, scale=WIDE ** -0.5), dtp=r(WIDE, RANK, scale=RANK ** -0.5), dt_bias=r(WIDE) - 3.0,
                A_log=torch.log(torch.arange(1, STATES + 1, dtype=torch.float64)).repeat(WIDE, 1), D=1 + r(WIDE, scale=0.1),
                norm=1 + r(WIDE, scale=0.1), out=r(HIDDEN, WIDE, scale=WIDE ** -0.5))


def layer(ops, w, x, marks=None, conv_state=None, state=None, **given):
    """One pass; `given`: where the new states go."""
    proj = x @ w["inp"].t()
    u, z = proj[..., :WIDE], proj[..., WIDE:]
    kw = {"state_out": given["conv_out"]} if given else {}
    u, conv_state = ops.causal_conv(u, w["conv"], w["conv_bias"], conv_state, activation="silu", starts=marks, **kw)
    p = u @ w["xp"].t()
    dt, B, C = p[..., :RANK] @ w["dtp"].t(), p[..., RANK:RANK + STATES], p[..., RANK + STATES:]
    kw = {"state_out": given["state_out"]} if given else {}
    if ops is O:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    y, state = ops.selective_scan(u, dt, -torch.exp(w["A_log"]), B, C, w["D"], dt_bias=w["dt_bias"], state=state, starts=marks, **kw)
    y = ops.group_norm(y, HEADS, w["norm"], None, gate=z, activation="silu")
    return y @ w["out"].t(), conv_state, state


def on_gpu(w, grad=False):
    return {k: v.float().cuda().requires_grad_(grad) for k, v in w.items()}


def batch(B, T, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, HIDDEN, generator=g, dtype=torch.float64)
    marks = torch.rand(B, T, generator=g) < 0.05
    return x, marks


def test_training():
    x, marks = batch(3, 70)
    w = weights()
    ref = {k: v.clone().requires_grad_() for k, v in w.items()}
    want, _, _ = layer(O, ref, x, marks)
    up = torch.randn(want.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    exp = torch.autograd.grad(want, list(ref.values()), up)
    dev = on_gpu(w, grad=True)
    got, _, _ = layer(tb, dev, x.float().cuda(), marks.cuda())
    # a norm divides by its heads' deviations, 16 features each: errors of the scan relative to a head's scale, not the tensor's
    close(got, want, "y", 2.0 ** -12)
    for a, b, n in zip(torch.autograd.grad(got, list(dev.values()), up.float().cuda()), exp, w):
        close(a, b, n, 2.0 ** -11)


def test_sequences_padded_on_the_left_and_generation():
    """Prompts of 5, 12 and 9 tokens in one batch, a start where each begins; then token by token, the states where they lie, against
    every sequence on its own."""
    w = weights()
    dev = on_gpu(w)
    lengths, T, more = (5, 12, 9), 12, 6
    g = torch.Generator().manual_seed(4)
    seqs = [torch.randn(1, n + more, HIDDEN, generator=g, dtype=torch.float64) for n in lengths]
    wants = [layer(O, w, s)[0] for s in seqs]
    x = torch.full((3, T, HIDDEN), 0.3, dtype=torch.float64)  # (whatever the padding holds)
    marks = torch.zeros(3, T, dtype=torch.bool)
    for i, (s, n) in enumerate(zip(seqs, lengths)):
        x[i, T - n:] = s[0, :n]
        marks[i, T - n] = True
    with torch.no_grad():
        y, conv_state, state = layer(tb, dev, x.float().cuda(), marks.cuda())
        for i, n in enumerate(lengths):
            close(y[i, T - n:], wants[i][0, :n], f"prompt {i}", 2.0 ** -12)
        step = lambda x: layer(tb, dev, x, None, conv_state, state, conv_out=conv_state, state_out=state)[0]  # noqa: E731
        token = torch.zeros(3, 1, HIDDEN, device="cuda")
        keep = conv_state.clone(), state.clone()
        step(token)  # (warm-up outside the capture; the states back)
        conv_state.copy_(keep[0]), state.copy_(keep[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(token)
        for t in range(more):
            token.copy_(torch.cat([s[:, n + t:n + t + 1] for s, n in zip(seqs, lengths)]))
            graph.replay()
            for i, n in enumerate(lengths):
                close(out[i, 0], wants[i][0, n + t], f"token {t} of {i}", 2.0 ** -12)


def test_two_captured_generations_share_nothing():
    """Two graphs of the same step, each with states of its own, replayed in turn on two streams."""
    w = on_gpu(weights())
    x = torch.randn(2, 1, HIDDEN, device="cuda")
    states = [(torch.randn(2, 3, WIDE, device="cuda"), torch.randn(2, WIDE, STATES, device="cuda")) for _ in range(2)]
    starts = [(a.clone(), b.clone()) for a, b in states]
    with torch.no_grad():
        layer(tb, w, x)
        graphs, outs = [], []
        for c, s in states:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(layer(tb, w, x, None, c, s, conv_out=c, state_out=s)[0])
            graphs.append(g)
        streams = [torch.cuda.Stream() for _ in graphs]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for (c0, s0), (c, s), out in zip(starts, states, outs):
            for _ in range(3):
                want, c0, s0 = layer(tb, w, x, None, c0, s0)
            assert torch.equal(c, c0) and torch.equal(s, s0) and torch.equal(out, want)
