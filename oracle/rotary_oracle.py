"""Rotary positions and the norm of queries and keys in float64 on the CPU, from their definitions."""

from __future__ import annotations

import math

import torch


def angles(cfg, positions):
    """positions [..] (integers) -> angles [.., rotary_dim / 2] and what the rotated features are multiplied by."""
    r, out, size = cfg.rotary_dim or cfg.head_dim, [], 1.0
    for p in range(r // 2):
        f = math.exp(-2.0 * p / r * math.log(cfg.theta))
        if cfg.scaling == "linear":
            f = f / cfg.factor
        elif cfg.scaling == "ntk":
            f = math.exp(-2.0 * p / r * (math.log(cfg.theta) + r / (r - 2) * math.log(cfg.factor)))
        elif cfg.scaling == "by_parts":
            turns = cfg.original_length / (2 * math.pi / f)
            if turns < cfg.beta_slow:
                f = f / cfg.factor
            elif turns <= cfg.beta_fast:
                keep = (turns - cfg.beta_slow) / (cfg.beta_fast - cfg.beta_slow)
                f = (1 - keep) * f / cfg.factor + keep * f
            size = 0.1 * math.log(cfg.factor) + 1.0
        out.append(f)
    pos = positions % cfg.wrap if cfg.wrap else positions
    return pos[..., None].double() * torch.tensor(out, dtype=torch.float64), size


def rotate(x, cfg, positions):
    """x [B,H,T,F], positions [T] or [B,T]."""
    r = cfg.rotary_dim or cfg.head_dim
    a, size = angles(cfg, positions)
    a = a[None, None] if a.dim() == 2 else a[:, None]
    c, s = a.cos() * size, a.sin() * size
    first = torch.arange(0, r, 2) if cfg.layout == "interleaved" else torch.arange(r // 2)
    second = first + (1 if cfg.layout == "interleaved" else r // 2)
    one, two = x[..., first], x[..., second]
    cols = [None] * x.shape[-1]
    for n, (i, j) in enumerate(zip(first.tolist(), second.tolist())):
        cols[i] = one[..., n] * c[..., n] - two[..., n] * s[..., n]
        cols[j] = two[..., n] * c[..., n] + one[..., n] * s[..., n]
    return torch.stack([x[..., i] if v is None else v for i, v in enumerate(cols)], -1)


def norm(x, w=None, eps=1e-6):
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return y if w is None else y * w
