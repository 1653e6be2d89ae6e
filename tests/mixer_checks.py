"""Comparing results of the selective layer's operators with their float64 oracle.

A result of type t is off by its rounding, at most finfo(t).eps / 2 of its value, and by the float32 arithmetic before it.
The latter is bounded relative to the tensor's scale (its root mean square): a handful of float32 operations and approximate
exponentials and quotients (2^-21 each) stay below 2^-16 of it; sums of n terms that do not agree in sign add n 2^-24 of
their own scale, 2^-13 for the n <= 2^11 of these tests."""

import torch

ELEMENT, SUM = 2.0 ** -16, 2.0 ** -13


def close(got, want, name, arithmetic=ELEMENT):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    g, w = got.detach().double().cpu(), want.detach().double().cpu()
    assert torch.equal(torch.isfinite(g), torch.isfinite(w)), name
    scale = w.pow(2).mean().sqrt()
    bound = torch.finfo(got.dtype).eps / 2 * w.abs() + arithmetic * (scale + w.abs())
    off = (g - w).abs() - bound
    assert (off <= 0).all(), f"{name}: {(off > 0).sum()} of {w.numel()} outside, worst {off.max():.3g} beyond the bound, scale {scale:.3g}"


def leaves(tensors, device="cuda"):
    """(leaves on the device, the same values in float64 as leaves on the CPU); None stays None."""
    def leaf(t, *to):
        return t.detach().to(*to).requires_grad_() if t.is_floating_point() else t.to(to[0])
    return ([None if t is None else leaf(t, device) for t in tensors],
            [None if t is None else leaf(t, "cpu", torch.float64) if t.is_floating_point() else t for t in tensors])


def grads(outs, ins, gs):
    ins = [t for t in ins if t is not None and t.is_floating_point()]
    return torch.autograd.grad(outs, ins, gs)
