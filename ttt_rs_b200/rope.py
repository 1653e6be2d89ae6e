"""Rotary positions and the norm of queries and keys (csrc/ttt_rotary.cu), for layers that place their heads otherwise than the
reference does (neighbouring pairs over the whole head, unscaled: rust/core/src/util.rs:284-392): pairs of either layout, a part
of the head, angles scaled for contexts longer than the trained ones, any positions; and a root-mean-square norm of every
head's query and key in the same pass.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch

from . import _lib
from ._lib import TttError
from .fused import _expect, device_status

_SCALINGS = ("none", "linear", "ntk", "by_parts")


@dataclass(frozen=True)
class RotaryConfig:
    """Pair p of the first `rotary_dim` (None: all) features of a head turns by position * theta^(-2p / rotary_dim).

    layout    "interleaved": features (2p, 2p + 1) are a pair, as in the layer; "half": (p, p + rotary_dim / 2)
    scaling   for contexts `factor` times as long as `original_length`:
              "linear"    every frequency divided by factor (positions interpolated)
              "ntk"       theta multiplied by factor^(rotary_dim / (rotary_dim - 2)): the slowest pair as in "linear"
              "by_parts"  pairs that turn less than `beta_slow` times over original_length as in "linear", those that turn more
                          than `beta_fast` times as they are, linearly between; results grow by 0.1 ln(factor) + 1
                          (arXiv:2309.00071)
    wrap      > 0: positions modulo this (the layer's "rope": the mini-batch)"""
    head_dim: int
    rotary_dim: Optional[int] = None
    theta: float = 10000.0
    layout: str = "interleaved"
    scaling: str = "none"
    factor: float = 1.0
    original_length: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    wrap: int = 0

    def __post_init__(self):
        r = self.width
        if self.head_dim < 2 or self.head_dim > 256 or self.head_dim % 2:
            raise ValueError(f"head_dim must be even, 2..256 (got {self.head_dim})")
        if r < 2 or r > self.head_dim or r % 2:
            raise ValueError(f"rotary_dim must be even, 2..head_dim (got {r})")
        if not self.theta >= 1.0 or not math.isfinite(self.theta):
            raise ValueError(f"theta must be at least 1 (got {self.theta})")
        if self.layout not in ("interleaved", "half"):
            raise ValueError(f"layout must be 'interleaved' or 'half' (got {self.layout!r})")
        if self.scaling not in _SCALINGS:
            raise ValueError(f"scaling must be one of {_SCALINGS} (got {self.scaling!r})")
        if self.scaling != "none" and not (self.factor >= 1.0 and math.isfinite(self.factor)):
            raise ValueError(f"factor must be at least 1 (got {self.factor})")
        if self.scaling == "ntk" and r < 4:
            raise ValueError("'ntk' needs a rotary_dim of at least 4")
        if self.scaling == "by_parts" and not (self.original_length > 0 and self.beta_fast > self.beta_slow >= 0.0):
            raise ValueError("'by_parts' needs original_length > 0 and beta_fast > beta_slow >= 0")
        if self.wrap < 0:
            raise ValueError(f"wrap must not be negative (got {self.wrap})")

    @property
    def width(self) -> int:
        return self.head_dim if self.rotary_dim is None else self.rotary_dim

    @property
    def size(self) -> float:
        """What the rotated features are multiplied by."""
        return 0.1 * math.log(self.factor) + 1.0 if self.scaling == "by_parts" else 1.0

    def frequencies(self) -> List[float]:
        """Radians per position of every pair."""
        r = self.width
        theta = self.theta * self.factor ** (r / (r - 2)) if self.scaling == "ntk" else self.theta
        out = []
        for p in range(r // 2):
            f = theta ** (-2.0 * p / r)
            if self.scaling == "linear":
                f /= self.factor
            elif self.scaling == "by_parts":
                turns = self.original_length * f / (2.0 * math.pi)
                keep = min(1.0, max(0.0, (turns - self.beta_slow) / (self.beta_fast - self.beta_slow)))
                f *= keep + (1.0 - keep) / self.factor
            out.append(f)
        return out


class Rotary:
    """A configuration with its table on a device: what a program makes once and hands to every call there."""

    def __init__(self, config: RotaryConfig, device=None):
        self.config = config
        self.device = torch.device("cuda" if device is None else device)
        # turns per position in 2^-64, as the kernels multiply them (modulo one turn, so that sign does not matter)
        turns = [round(f / (2.0 * math.pi) * 2.0 ** 64) for f in config.frequencies()]
        with torch.inference_mode(False):  # (a table made while serving is saved for the backward of a later call)
            self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64, device=self.device)
        self._args = (self.turns, config.width, int(config.layout == "half"), config.wrap, config.size)


_NO_ROTATION = (None, 0, 0, 0, 1.0)


def _check_heads(name: str, x: torch.Tensor, F: Optional[int] = None):
    if not x.is_cuda:
        raise TttError(_lib.TTT_ERR_CUDA, "inputs must be CUDA tensors: this operator has no CPU path")
    if x.dim() != 4:
        raise TttError(_lib.TTT_ERR_SHAPE, f"{name} must be [batch, heads, seq_len, head_dim], got {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TttError(_lib.TTT_ERR_UNSUPPORTED, f"unsupported dtype {x.dtype}")
    if x.numel() == 0:
        raise TttError(_lib.TTT_ERR_SHAPE, "batch, heads and seq_len must be positive")
    if F is not None and x.shape[3] != F:
        raise TttError(_lib.TTT_ERR_SHAPE, f"{name} has head_dim {x.shape[3]}, the rotation {F}")


def _check_positions(positions: Optional[torch.Tensor], B: int, T: int, device):
    if positions is None:
        return None
    if positions.dtype not in (torch.int32, torch.int64):
        raise TttError(_lib.TTT_ERR_SHAPE, f"positions must be int32 or int64 (got {positions.dtype})")
    if tuple(positions.shape) not in ((T,), (1, T), (B, T)):
        raise TttError(_lib.TTT_ERR_SHAPE, f"positions has shape {tuple(positions.shape)}, expected {(T,)} or {(B, T)}")
    if positions.device != device:
        raise TttError(_lib.TTT_ERR_SHAPE, f"positions is on {positions.device}, expected {device}")
    return positions.long().contiguous()


def _check_out(out, like, name: str, *others: Optional[torch.Tensor]):
    """`others`: what else the call reads or writes."""
    if out is None:
        return
    _expect(name, out, like.shape, like.dtype, like.device)
    if out.shape[3] > 1 and out.stride(3) != 1:
        raise TttError(_lib.TTT_ERR_SHAPE, f"rows of {name} must be contiguous")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (out, like, *others)):
        raise TttError(_lib.TTT_ERR_UNSUPPORTED, "results that are given are not recorded for autograd")


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if x.shape[3] == 1 or x.stride(3) == 1 else x.contiguous()


def _check_table(rot: Rotary, device):
    if rot.turns.device != device:
        raise TttError(_lib.TTT_ERR_SHAPE, f"the rotation's table is on {rot.turns.device}, the tensors on {device}")


def rotary(x: torch.Tensor, rot: Rotary, start_idx: int = 0, positions: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [B,H,T,F] (float32 or bfloat16, head_dim even up to 256; any strides with contiguous rows: [B,T,H,F] and columns of a
    projection as views) with its rows rotated to positions start_idx + t, or to `positions` ([T] or [B,T], int32 or int64, of
    either sign).  The result is contiguous [B,H,T,F], or `out` (which may be x itself but share no other element with it; not recorded
    for autograd, and refused where that asks for gradients).  Differentiable with respect to x, once and not in forward mode."""
    native = _lib.host().rotary(x, *rot._args, positions, start_idx, 0, out) if isinstance(x, torch.Tensor) and \
        x.dim() == 4 and x.shape[3] == rot.config.head_dim else None
    if native is not None:
        return native
    _check_heads("x", x, rot.config.head_dim)
    _check_table(rot, x.device)
    _check_out(out, x, "out")
    positions = _check_positions(positions, x.shape[0], x.shape[2], x.device)
    device_status(x.device)
    native = _lib.host().rotary(_rows(x), *rot._args, positions, start_idx, 0, out)
    if native is None:
        raise TttError(_lib.TTT_ERR_SHAPE, _lib.last_error() or "unsupported problem for the rotation")
    return native


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None, rot: Optional[Rotary] = None, eps: float = 1e-6, start_idx: int = 0,
                   positions: Optional[torch.Tensor] = None,
                   out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Every head's query and key divided by its root mean square, sqrt(mean(x^2) + eps), multiplied by the weight ([F], of the
    inputs' type; None: ones) and rotated (`rot` None: not), in one pass over both.  q [B,H,T,F] and k [B,Hk,T,F] as in `rotary`,
    Hk of any number; results contiguous [B,H,T,F], [B,Hk,T,F], or `out` as in `rotary` (each may be its own input; neither may share
    elements with the other's or with the other result).  Differentiable with respect to q, k and the weights, as `rotary` is."""
    args = _NO_ROTATION if rot is None else rot._args
    oq, ok = (None, None) if out is None else out
    fits = rot is None or (isinstance(q, torch.Tensor) and q.dim() == 4 and q.shape[3] == rot.config.head_dim)
    native = _lib.host().qk_norm(q, k, q_weight, k_weight, *args, positions, start_idx, eps, oq, ok) if fits else None
    if native is not None:
        return native
    F = None if rot is None else rot.config.head_dim
    _check_heads("q", q, F)
    _check_heads("k", k, F)
    B, _, T, F = q.shape
    _expect("k", k, (B, k.shape[1], T, F), q.dtype, q.device)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            _expect(name, w, (F,), q.dtype, q.device)
    if rot is not None:
        _check_table(rot, q.device)
    _check_out(oq, q, "out[0]", k, q_weight, k_weight)
    _check_out(ok, k, "out[1]", q, q_weight, k_weight)
    positions = _check_positions(positions, B, T, q.device)
    device_status(q.device)
    native = _lib.host().qk_norm(_rows(q), _rows(k), None if q_weight is None else q_weight.contiguous(),
                                 None if k_weight is None else k_weight.contiguous(), *args, positions, start_idx, eps, oq, ok)
    if native is None:
        raise TttError(_lib.TTT_ERR_SHAPE, _lib.last_error() or "unsupported problem for the norm and rotation")
    return native
