"""Selective state space scan whose sequences are cut into segments, for every padded number of states, against its oracle;
narrow groups over many tokens; gradients that are strided; offsets behind 32 bits in gradients."""

import pytest
import torch

import ttt_rs_b200 as tb
from mixer_checks import ELEMENT, SUM, close, grads, leaves
from oracle import mixer_oracle as O
from test_selective_scan_gpu import NAMES, make, scan
from ttt_rs_b200 import _lib

pytestmark = pytest.mark.gpu

CASES = [  # B, T, C, N, G: the first row of each has no start, the last one has some
    (2, 700, 12, 3, 3), (2, 333, 40, 4, 2), (2, 500, 24, 8, 2), (2, 650, 24, 16, 4), (2, 410, 20, 32, 2), (2, 330, 12, 64, 3), (2, 300, 10, 33, 2),
    (1, 700, 48, 16, 8), (9, 200, 5, 16, 1),  # narrow groups, few channels
    (19, 200, 48, 16, 8), (19, 200, 48, 4, 8), (19, 200, 48, 64, 8),  # 152 blocks
]


def floats_of_one_segment(B, T, C, N, G):
    """The backward's workspace for sequences in one piece: shares of dB and dC, of dA, of dD and the bias's gradient."""
    padded = max(4, 1 << (N - 1).bit_length())
    blocks = -(-(C // G) // {4: 128, 8: 64}.get(padded, 1024 // padded))
    return B * G * blocks * T * 2 * padded + B * C * padded + (2 * B * C + 3) // 4 * 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_results_and_gradients(case, dtype):
    B, T, C, N, G = case
    lib, shape = _lib.load(), (B, T, C, G, N, _lib.TTT_BF16 if dtype == torch.bfloat16 else _lib.TTT_F32)
    assert lib.ttt_linear_selective_forward_workspace_bytes(*shape) > 0  # (several segments)
    assert lib.ttt_linear_selective_backward_workspace_bytes(*shape) > 4 * floats_of_one_segment(*case)
    ins, marks = make(B, T, C, N, G, dtype, seed=T + C)
    dev, ref = leaves(ins)
    outs, want = scan(tb.selective_scan, dev, marks.cuda()), scan(O.selective_scan, ref, marks)
    for o, w, n in zip(outs, want, ("y", "state")):
        close(o, w, n, 2 * ELEMENT)
    g = torch.Generator().manual_seed(7)
    up = [torch.randn(w.shape, generator=g).to(o.dtype) for w, o in zip(want, outs)]
    got, exp = grads(outs, dev, [u.cuda() for u in up]), grads(want, ref, [u.double() for u in up])
    # sums of B T terms: n 2^-24 of their scale
    for a, b, n in zip(got, exp, NAMES):
        close(a, b, n, SUM if B * T <= 2048 else 2 * SUM)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strided_gradients(dtype):
    """Gradients of the results that lie in wider rows, with batch and token exchanged, or with channels apart."""
    ins, marks = make(2, 70, 32, 16, 1, dtype)
    dev = [t.cuda().requires_grad_() for t in ins]
    on = marks.cuda()
    conv = [dev[0], torch.randn(32, 4, device="cuda").to(dtype).requires_grad_()]
    gy, gs = torch.randn(2, 70, 32, device="cuda").to(dtype), torch.randn(2, 32, 16, device="cuda")
    wide = torch.zeros(2, 70, 53, device="cuda", dtype=dtype)
    wide[..., 3:35] = gy
    given = [wide[..., 3:35], gy.transpose(0, 1).contiguous().transpose(0, 1), gy.transpose(1, 2).contiguous().transpose(1, 2)]
    turned = gs.transpose(1, 2).contiguous().transpose(1, 2)
    want = grads(scan(tb.selective_scan, dev, on), dev, [gy, gs])
    want_conv = grads(tb.causal_conv(*conv, activation="silu", starts=on)[0], conv, gy)
    for v, s in zip(given, (gs, turned, turned)):
        assert torch.equal(v, gy) and torch.equal(s, gs)
        for a, b, n in zip(grads(scan(tb.selective_scan, dev, on), dev, [v, s]), want, NAMES):
            assert torch.equal(a, b), n
        got = grads(tb.causal_conv(*conv, activation="silu", starts=on)[0], conv, v)
        # (rows off a vector's address are walked by other threads: sums in another order, one rounding apart)
        assert torch.equal(got[0], want_conv[0])
        close(got[1], want_conv[1], "weight", torch.finfo(dtype).eps + SUM)
    one = torch.ones(1, 1, 1, device="cuda", dtype=dtype).expand(2, 70, 32)
    for a, b in zip(grads(scan(tb.selective_scan, dev, on)[0], dev, one), grads(scan(tb.selective_scan, dev, on)[0], dev, one.contiguous())):
        assert torch.equal(a, b)


def test_gradients_behind_32_bits():
    """Tensors of more than 2^31 elements: the last tokens' gradients."""
    T, C = 70000, 32768
    r = lambda *s: torch.randn(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    x = torch.zeros(1, T, C, device="cuda", dtype=torch.bfloat16)
    x[0, -4:] = r(4, C)
    gy = torch.zeros(1, T, C, device="cuda", dtype=torch.bfloat16)
    gy[0, -2:] = r(2, C)
    w, last = r(C, 4), slice(T - 8, T)
    few, few_gy = x[:, last].double().cpu().requires_grad_(), gy[:, last].double().cpu()
    x.requires_grad_()
    w.requires_grad_()
    gx, gw = torch.autograd.grad(tb.causal_conv(x, w)[0], (x, w), gy)
    wr = w.detach().double().cpu().requires_grad_()
    ex, ew = torch.autograd.grad(O.causal_conv(few, wr)[0], (few, wr), few_gy)
    close(gx[:, last], ex, "convolution, x")
    close(gw, ew, "convolution, weight", SUM)
    assert not gx[0, :-8].any()
    del gx
    scale = (1 + 0.1 * r(C)).requires_grad_()
    gx, gw = torch.autograd.grad(tb.group_norm(x, 512, scale, eps=1e-3), (x, scale), gy)
    wr = scale.detach().double().cpu().requires_grad_()
    ex, ew = torch.autograd.grad(O.group_norm(few, 512, wr, eps=1e-3), (few, wr), few_gy)
    close(gx[:, last], ex, "norm, x", 4 * ELEMENT)
    close(gw, ew, "norm, weight", SUM)
    assert not gx[0, :-8].any()
    del gx
    # steps of log 2, rates of -1: a token halves what was before it
    dt = torch.zeros(1, 1, C, device="cuda", dtype=torch.bfloat16).expand(1, T, C)
    A = torch.full((C, 4), -1.0, device="cuda")
    b = torch.ones(1, T, 4, device="cuda", dtype=torch.bfloat16)
    (gx,) = torch.autograd.grad(tb.selective_scan(x, dt, A, b, b)[0], x, gy)
    zero, one = torch.zeros(1, 8, C, dtype=torch.float64), torch.ones(1, 8, 1, 4, dtype=torch.float64)
    (ex,) = torch.autograd.grad(O.selective_scan(few, zero, A.double().cpu(), one, one)[0], few, few_gy)
    close(gx[:, last], ex, "scan, x", 2 * ELEMENT)
    assert gx[0, :64].abs().max() == 0  # (2^-70000 of a gradient)
