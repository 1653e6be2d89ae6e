"""Oracles of the operators of a selective state space layer, token by token in float64, differentiable by autograd: causal
convolution, selective scan, group norm with channels last.  The tests compare the CUDA kernels' results with these (the
formulas: csrc/ttt_conv.cu, csrc/ttt_selective.cuh, csrc/ttt_norm.cu)."""

import math

import torch


def act(v, name):
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def causal_conv(x, weight, bias=None, state=None, activation=None, starts=None):
    """x [B,T,C], weight [C,K], state [B,K-1,C], starts [B,T] -> (y [B,T,C], new state)."""
    B, T, C = x.shape
    K = weight.shape[1]
    window = list(torch.zeros(K - 1, B, C, dtype=x.dtype).unbind()) if state is None else list(state.unbind(1))
    out = []
    for t in range(T):
        if starts is not None:
            window = [torch.where(starts[:, t, None], torch.zeros_like(w), w) for w in window]
        window.append(x[:, t])
        v = sum(w * weight[:, j] for j, w in enumerate(window))
        out.append(act(v if bias is None else v + bias, activation))
        window = window[1:]
    return torch.stack(out, 1), torch.stack(window, 1)


def selective_scan(x, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, state=None, softplus=True, starts=None):
    """x, dt, z [B,T,C]; A [C,N]; Bm, Cm [B,T,G,N]; D, dt_bias [C]; state [B,C,N] -> (y [B,T,C], new state)."""
    B, T, C = x.shape
    G, N = Bm.shape[2:]
    h = torch.zeros(B, C, N, dtype=x.dtype) if state is None else state
    wide = lambda t: t.repeat_interleave(C // G, 1)  # noqa: E731
    out = []
    for t in range(T):
        v = dt[:, t] if dt_bias is None else dt[:, t] + dt_bias
        d = torch.nn.functional.softplus(v, threshold=1e9) if softplus else v
        if starts is not None:
            h = torch.where(starts[:, t, None, None], torch.zeros_like(h), h)
        h = torch.exp(d[..., None] * A) * h + (d * x[:, t])[..., None] * wide(Bm[:, t])
        y = (h * wide(Cm[:, t])).sum(-1)
        if D is not None:
            y = y + D * x[:, t]
        out.append(y if z is None else y * act(z[:, t], "silu"))
    return torch.stack(out, 1), h


def group_norm(x, groups, weight=None, bias=None, gate=None, activation=None, eps=1e-5, over="token"):
    g = x.unflatten(-1, (groups, -1))
    dims = (3,) if over == "token" else (1, 3)
    d = g - g.mean(dims, keepdim=True)
    u = (d / torch.sqrt((d * d).mean(dims, keepdim=True) + eps)).flatten(2)
    if weight is not None:
        u = u * weight
    if bias is not None:
        u = u + bias
    return act(u, activation) if gate is None else u * act(gate, activation)
