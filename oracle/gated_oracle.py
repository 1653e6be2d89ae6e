"""Gated linear recurrence token by token, in the inputs' precision (float64 for the tests).

    W_t = exp(g_t) W_{t-1} + beta_t k_t^T v_t,      o_t = q_t W_t
"""

from __future__ import annotations

import torch


def gated_forward(q, k, v, g, beta=None, w=None):
    """q, k, v [B,H,T,F], g and beta [B,H,T], w [B,H,F,F] -> (o [B,H,T,F], w behind the last token)."""
    B, H, T, F = q.shape
    w = torch.zeros(B, H, F, F, dtype=q.dtype) if w is None else w
    a = torch.exp(g)
    outs = []
    for t in range(T):
        kt = k[:, :, t] if beta is None else beta[:, :, t, None] * k[:, :, t]
        w = a[:, :, t, None, None] * w + kt[..., :, None] * v[:, :, t, None, :]
        outs.append((q[:, :, t, None, :] @ w)[:, :, 0])
    return torch.stack(outs, 2), w


def gated_grads(q, k, v, g, beta, w, d_out, d_w=None):
    """(o, w', gradients of q, k, v, g, beta, w for <d_out, o> + <d_w, w'>); None in the place of an absent input."""
    leaves = [None if t is None else t.detach().clone().requires_grad_() for t in (q, k, v, g, beta, w)]
    o, wn = gated_forward(*leaves)
    loss = (o * d_out).sum() + (0.0 if d_w is None else (wn * d_w).sum())
    have = [t for t in leaves if t is not None]
    got = iter(torch.autograd.grad(loss, have))
    return [o.detach(), wn.detach()] + [None if t is None else next(got) for t in leaves]


def gated_magnitudes(q, k, v, g, beta, w, d_out=None, d_w=None):
    """The same with every input's absolute value (g as it is): the sum of the absolute values of all terms that a result
    consists of, which is what roundings of factors and of partial sums are relative to."""
    a = [None if t is None else t.abs() for t in (q, k, v, beta, w, d_out, d_w)]
    if d_out is None:
        return list(gated_forward(a[0], a[1], a[2], g, a[3], a[4]))
    return gated_grads(a[0], a[1], a[2], g, a[3], a[4], a[5], a[6])
