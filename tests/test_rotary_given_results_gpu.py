"""Results of the rotary operators that are given: where they may lie, and what autograd knows of them."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def refused(code, call):
    import ttt_rs_b200 as tb
    with pytest.raises(tb.TttError) as e:
        call()
    assert e.value.code == code


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_that_share_elements_are_refused(dtype):
    """Views that are not dense: shifted by a token of a padded cache, by features of a projection."""
    import ttt_rs_b200 as tb
    from ttt_rs_b200 import _lib as L
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda")
    cache = torch.randn(2, 3, 50, 64, device="cuda").to(dtype)
    proj = torch.randn(2, 40, 4 * 3 * 64, device="cuda").to(dtype)
    was = cache.clone(), proj.clone()
    cols = lambda at: proj[..., at:at + 192].unflatten(-1, (3, 64)).transpose(1, 2)  # noqa: E731
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(cache[:, :, :40], rot, out=cache[:, :, 1:41]))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(cache[:, :, 1:41], rot, out=cache[:, :, :40]))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(cols(0), rot, out=cols(8)))
    refused(L.TTT_ERR_SHAPE, lambda: tb.qk_norm_rotary(cols(0), cols(192), rot=rot, out=(cols(384), cols(384 + 8))))
    refused(L.TTT_ERR_SHAPE, lambda: tb.qk_norm_rotary(cols(0), cols(192), rot=rot, out=(cols(192), cols(384))))
    assert torch.equal(cache, was[0]) and torch.equal(proj, was[1])
    # columns that share none, and the same rows: as apart from one another
    want = tb.qk_norm_rotary(cols(0), cols(192), rot=rot)
    tb.qk_norm_rotary(cols(0), cols(192), rot=rot, out=(cols(384), cols(576)))
    assert torch.equal(cols(384), want[0]) and torch.equal(cols(576), want[1])
    tb.qk_norm_rotary(cols(0), cols(192), rot=rot, out=(cols(0), cols(192)))
    assert torch.equal(cols(0), want[0]) and torch.equal(cols(192), want[1])
    want = tb.rotary(cache[:, :, 40:], rot)
    tb.rotary(cache[:, :, 40:], rot, out=cache[:, :, 5:15])
    assert torch.equal(cache[:, :, 5:15], want)


def test_results_that_require_gradients_are_refused():
    """As those of inputs and weights that do: nothing given is recorded."""
    import ttt_rs_b200 as tb
    from ttt_rs_b200 import _lib as L
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda")
    x, k, leaf = torch.randn(3, 2, 3, 8, 64, device="cuda")
    leaf = leaf.clone().requires_grad_()
    part, was, w = leaf * 1.0, leaf.detach().clone(), torch.ones(64, device="cuda").requires_grad_()
    for out in (leaf, part):
        refused(L.TTT_ERR_UNSUPPORTED, lambda: tb.rotary(x, rot, out=out))
        refused(L.TTT_ERR_UNSUPPORTED, lambda: tb.qk_norm_rotary(x, k, rot=rot, out=(out, torch.empty_like(k))))
        refused(L.TTT_ERR_UNSUPPORTED, lambda: tb.qk_norm_rotary(x, k, rot=rot, out=(torch.empty_like(x), out)))
    refused(L.TTT_ERR_UNSUPPORTED, lambda: tb.qk_norm_rotary(x, k, w, None, rot=rot, out=(torch.empty_like(x), torch.empty_like(k))))
    refused(L.TTT_ERR_UNSUPPORTED, lambda: tb.qk_norm_rotary(x, leaf, rot=rot, out=(torch.empty_like(x), torch.empty_like(k))))
    assert torch.equal(leaf.detach(), was) and torch.equal(part.detach(), was)
    with torch.no_grad():  # (as torch's own operations into a leaf)
        tb.rotary(x, rot, out=leaf)
        assert torch.equal(leaf, tb.rotary(x, rot))


def test_what_was_saved_and_is_overwritten_has_no_gradients():
    """Results written over a tensor that a graph has saved: its backward refuses, as it does after torch's own operations."""
    import ttt_rs_b200 as tb
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda")
    x, k, leaf = torch.randn(3, 2, 3, 8, 64, device="cuda")
    leaf.requires_grad_()
    calls = [lambda a: tb.rotary(a, rot, out=a), lambda a: tb.rotary(x, rot, out=a), lambda a: tb.rotary(x[:, :, :4], rot, out=a[:, :, 4:]),
             lambda a: tb.qk_norm_rotary(a, k, rot=rot, out=(a, k)), lambda a: tb.qk_norm_rotary(k, a, rot=rot, out=(k, a))]
    for call in calls:
        a = leaf.exp()  # (saves its result)
        before = a._version
        with torch.no_grad():
            call(a)
        assert a._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(a.sum(), leaf)
    a = leaf.exp()
    with torch.no_grad():
        y = tb.rotary(a, rot)
    assert y._version == 0 and torch.equal(torch.autograd.grad(a.sum(), leaf)[0], a.detach())
    with torch.inference_mode():
        b = torch.empty_like(x)
    with torch.no_grad():  # (counts no versions)
        assert torch.equal(tb.rotary(x, rot, out=b), tb.rotary(x, rot))


def test_a_rotation_made_in_inference_mode_can_be_differentiated():
    import ttt_rs_b200 as tb
    with torch.inference_mode():
        rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda")
    x, w = torch.randn(1, 2, 8, 64, device="cuda").requires_grad_(), torch.ones(64, device="cuda").requires_grad_()
    (dx,) = torch.autograd.grad(tb.rotary(x, rot).sum(), x)
    assert torch.isfinite(dx).all() and all(torch.isfinite(t).all() for t in torch.autograd.grad(tb.qk_norm_rotary(x, x, w, w, rot)[0].sum(), (x, w)))


def test_given_results_in_inference_mode():
    import ttt_rs_b200 as tb
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda")
    x, out = torch.randn(2, 2, 3, 8, 64, device="cuda")
    leaf = torch.randn(2, 3, 8, 64, device="cuda").requires_grad_()
    a = leaf.exp()
    with torch.inference_mode():
        want = tb.rotary(x, rot)
        assert torch.equal(tb.rotary(x, rot, out=out), want)  # (an ordinary tensor, written while serving)
        made = torch.empty_like(x)
        assert torch.equal(tb.rotary(x, rot, out=made), want)
        tb.rotary(x, rot, out=a)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(a.sum(), leaf)
