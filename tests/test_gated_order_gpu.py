"""The gated recurrence's kernels reuse shared memory that threads have written for the copies of later chunks: runs of many
chunks per block, several launches at once on the card, have to repeat bit by bit and meet the oracle."""

import pytest
import torch

import test_gated_linear_gpu as G
from oracle import gated_oracle as O

pytestmark = pytest.mark.gpu
# streams in ranges of whole and cut streams, one block per stream, and streams in segments
SHAPES = [(25, 20, 640, 64), (10, 16, 1500, 64), (1, 2, 6000, 64), (12, 16, 1000, 32)]


def on_three_streams(call, times=4):
    """`call` on three streams at once, several times over; all that it returned."""
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    torch.cuda.synchronize()
    for _ in range(times):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("B,H,T,F", SHAPES)
def test_backwards_of_many_chunks_repeat(B, H, T, F):
    import ttt_rs_b200 as tb
    ins, d_out, d_w = G.make(B, H, T, F, torch.bfloat16, seed=31)
    dev, u, dw = [t.cuda() for t in ins], d_out.cuda(), d_w.cuda()

    def call():
        leaves = [t.detach().requires_grad_() for t in dev]
        out, w = tb.fused_gated_linear(*leaves)
        return [out.detach(), w.detach(), *torch.autograd.grad([out, w], leaves, [u, dw])]

    want = call()
    assert all(torch.equal(x, y) for got in on_three_streams(call) for x, y in zip(got, want))
    one = [t[:1, :1] for t in ins]
    args = (*G.f64(one), d_out[:1, :1].double(), d_w[:1, :1].double())
    G.check([t[:1, :1] for t in want], O.gated_grads(*args), O.gated_magnitudes(*args), torch.bfloat16)
    tb.check_status()


@pytest.mark.parametrize("B,H,T,F", SHAPES)
def test_forwards_of_many_chunks_repeat(B, H, T, F):
    import ttt_rs_b200 as tb
    ins, _, _ = G.make(B, H, T, F, torch.bfloat16, seed=32)
    dev = [t.cuda() for t in ins]

    def call():
        with torch.no_grad():
            return tb.fused_gated_linear(*dev)

    want = call()
    assert all(torch.equal(x, y) for got in on_three_streams(call) for x, y in zip(got, want))
    one = G.f64([t[:1, :1] for t in ins])
    G.check([t[:1, :1] for t in want], O.gated_forward(*one), O.gated_magnitudes(*one), torch.bfloat16)
    tb.check_status()
