"""Tangents of forward-mode differentiation: the gated recurrence and the rotary operators compute none, and say so."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import test_gated_linear_gpu as G

pytestmark = pytest.mark.gpu


def refused(call):
    import ttt_rs_b200 as tb
    from ttt_rs_b200 import _lib as L
    for grad in (False, True):
        with torch.set_grad_enabled(grad), pytest.raises(tb.TttError, match="forward mode") as e:
            call()
        assert e.value.code == L.TTT_ERR_UNSUPPORTED


@pytest.mark.parametrize("T", [1, 70])
def test_gated(T):
    import ttt_rs_b200 as tb
    dev = [t.cuda() for t in G.make(1, 2, T, 64, torch.float32)[0]]
    with fwd.dual_level():
        for i, t in enumerate(dev):
            args = list(dev)
            args[i] = fwd.make_dual(t, torch.ones_like(t))
            refused(lambda: tb.fused_gated_linear(*args))
        turned = fwd.make_dual(dev[0], torch.ones_like(dev[0])).transpose(1, 2).contiguous().transpose(1, 2)
        refused(lambda: tb.fused_gated_linear(turned, *dev[1:]))
        odd = fwd.make_dual(dev[3], torch.ones_like(dev[3])).expand(1, 2, T).flip(-1)
        refused(lambda: tb.fused_gated_linear(*dev[:3], odd, *dev[4:]))
    with torch.no_grad():
        tb.fused_gated_linear(*dev)


def test_rotary_and_norm():
    import ttt_rs_b200 as tb
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda")
    x, k = torch.randn(2, 2, 3, 8, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    with fwd.dual_level():
        dx, dw = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(w, torch.ones_like(w))
        refused(lambda: tb.rotary(dx, rot))
        refused(lambda: tb.rotary(dx[..., ::2], tb.Rotary(tb.RotaryConfig(head_dim=32), device="cuda")))  # (rows that are copied first)
        refused(lambda: tb.rotary(k, rot, out=dx))
        refused(lambda: tb.qk_norm_rotary(dx, k, rot=rot))
        refused(lambda: tb.qk_norm_rotary(k, dx, w, w, rot=rot))
        refused(lambda: tb.qk_norm_rotary(x, k, w, dw, rot=rot))
    assert torch.equal(tb.rotary(x, rot), tb.rotary(x, rot))
