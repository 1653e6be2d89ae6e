"""Operators of a layer that remembers through a selective state space scan, on [batch, seq_len, channels] with channels last:
its short causal convolution (csrc/ttt_conv.cu), the scan (csrc/ttt_selective*.cu) and the group norm with its gate
(csrc/ttt_norm.cu).  (The reference has none of them.)
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import TttError
from .fused import _expect

_CONV_ACTIVATIONS = {None: 0, "silu": 1}
_NORM_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}
_OVER = {"token": 0, "sequence": 1}


def _unknown(what: str, name, known) -> TttError:
    return TttError(_lib.TTT_ERR_UNSUPPORTED, f"{what} must be one of {tuple(known)} (got {name!r})")


def _check_rows(name: str, x: torch.Tensor):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TttError(_lib.TTT_ERR_CUDA, "inputs must be CUDA tensors: this operator has no CPU path")
    if x.dim() != 3:
        raise TttError(_lib.TTT_ERR_SHAPE, f"{name} must be [batch, seq_len, channels], got {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TttError(_lib.TTT_ERR_UNSUPPORTED, f"unsupported dtype {x.dtype}")
    if x.numel() == 0:
        raise TttError(_lib.TTT_ERR_SHAPE, "batch, seq_len and channels must be positive")


def _rows(x: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """x [B,T,C] as the kernels take it: contiguous channels."""
    return x if x is None or x.shape[2] == 1 or x.stride(2) == 1 else x.contiguous()


def _dense(x: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if x is None else x.contiguous()


def _aligned(x: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if x is None:
        return None
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _check_starts(starts: Optional[torch.Tensor], B: int, T: int, device):
    if starts is None:
        return
    if starts.dtype not in (torch.bool, torch.uint8):
        raise TttError(_lib.TTT_ERR_SHAPE, f"starts must be bool or uint8 (got {starts.dtype})")
    _expect("starts", starts, (B, T), starts.dtype, device)


def _check_state_out(out: Optional[torch.Tensor], shape, dtype, device, *inputs: Optional[torch.Tensor]):
    if out is None:
        return
    _expect("state_out", out, shape, dtype, device)
    if not out.is_contiguous():
        raise TttError(_lib.TTT_ERR_SHAPE, "state_out must be contiguous")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (out, *inputs)):
        raise TttError(_lib.TTT_ERR_UNSUPPORTED, "results that are given are not recorded for autograd")


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                activation: Optional[str] = None, starts: Optional[torch.Tensor] = None,
                state_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y [B,T,C], new state [B,K-1,C]) of the causal depthwise convolution y_t = act(bias + sum_j weight_j x_{t-K+1+j}), any number of
    tokens, single ones included.  x [B,T,C] (float32 or bfloat16; any strides that are not negative, with contiguous channels: columns
    of a projection are read where they lie), weight [C,K] with 2 to 4 taps, bias [C] (None: none) and state [B,K-1,C], the inputs before
    the first token (None: zeros), of x's type; activation None or "silu".  starts [B,T] (bool or uint8): a token with a start, and
    those behind it, see nothing before it, so that sequences may follow one another in one row, or be padded on the left (where not with
    finite numbers: the gradients of weight and bias sum over all tokens, and a gradient of zero times a NaN is one).  The new state
    is the last K-1 inputs as far as they are visible (zeros elsewhere), in `state_out` where given (it may be `state` itself but share
    nothing with another tensor; not recorded for autograd, and refused where that asks for gradients).  Differentiable with respect to
    x, weight, bias and state, through both results, once and not in forward mode; sums are float32."""
    act = _CONV_ACTIVATIONS.get(activation)
    if act is None:
        raise _unknown("activation", activation, _CONV_ACTIVATIONS)
    native = _lib.host().causal_conv(x, weight, bias, state, act, starts, state_out)
    if native is not None:
        return native
    _check_rows("x", x)
    B, T, C = x.shape
    if weight.dim() != 2 or not 2 <= weight.shape[1] <= 4:
        raise TttError(_lib.TTT_ERR_UNSUPPORTED, f"weight must be [channels, 2..4 taps], got {tuple(weight.shape)}")
    held = (B, weight.shape[1] - 1, C)
    _expect("weight", weight, (C, weight.shape[1]), x.dtype, x.device)
    if bias is not None:
        _expect("bias", bias, (C,), x.dtype, x.device)
    if state is not None:
        _expect("state", state, held, x.dtype, x.device)
    _check_starts(starts, B, T, x.device)
    _check_state_out(state_out, held, x.dtype, x.device, x, weight, bias, state)
    native = _lib.host().causal_conv(_rows(x), weight.contiguous(), _dense(bias), _dense(state), act, _dense(starts), state_out)
    if native is None:
        raise TttError(_lib.TTT_ERR_SHAPE, _lib.last_error() or "unsupported problem for the causal convolution")
    return native


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor] = None,
                   z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                   softplus: bool = True, starts: Optional[torch.Tensor] = None,
                   state_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y [B,T,C], state behind the last token [B,C,N] float32) of the selective state space scan

        d_t = softplus(dt_t + dt_bias),   h_t = exp(d_t A) h_{t-1} + d_t x_t B_t,   y_t = (<C_t, h_t> + D x_t) * SiLU(z_t)

    for every channel, any number of tokens; without gradients a call of up to 16 tokens runs as a decode step.  x, dt and z (None: no
    gate) [B,T,C], float32 or bfloat16, and B, C [B,T,G,N] or [B,T,N] (one group) of the same type, shared by the C / G neighbouring
    channels of a group: strides that are not negative, with contiguous channels and states (columns of a projection are read where they
    lie).  A [C,N], 1 to 64 states per channel, at most 0 for states that do not grow (-inf keeps nothing of a state, but a step
    of zero keeps all of it at any rate; rates below -2^100 / log2(e) count as that); D, dt_bias [C] (None: zeros); state [B,C,N], the
    state before the first token (None: zeros): float32.  softplus=False: d_t = dt_t + dt_bias.  starts [B,T] (bool or uint8): such a token
    finds a state of zero, so that sequences may follow one another in one row, or be padded on the left; nothing before it is seen, not
    even a NaN (the gradients of A, D and dt_bias sum over all tokens, though, and those of B and C over a group's channels: a gradient of
    zero times a NaN is one).  The new state goes to `state_out` where given (contiguous and on 16 bytes; it may be `state` itself but share
    nothing with another tensor; not recorded for autograd, and refused where that asks for gradients).  Differentiable with respect to all nine, through both results,
    once and not in forward mode.  Steps, decays, states and sums are float32, and results are rounded to bfloat16 once."""
    native = _lib.host().selective(x, dt, A, B, C, D, z, dt_bias, state, starts, softplus, state_out)
    if native is not None:
        return native
    _check_rows("x", x)
    b, T, ch = x.shape
    dev = x.device
    _expect("dt", dt, x.shape, x.dtype, dev)
    B, C = (t.unsqueeze(2) if t.dim() == 3 else t for t in (B, C))
    if B.dim() != 4 or ch % max(1, B.shape[2]) or B.numel() == 0:
        raise TttError(_lib.TTT_ERR_SHAPE, f"B must be [batch, seq_len, groups, states] with groups that divide {ch} channels, got {tuple(B.shape)}")
    G, N = B.shape[2:]
    if N > 64:
        raise TttError(_lib.TTT_ERR_UNSUPPORTED, f"Unsupported states={N} (supported: 1..64)")
    _expect("B", B, (b, T, G, N), x.dtype, dev)
    _expect("C", C, (b, T, G, N), x.dtype, dev)
    _expect("A", A, (ch, N), torch.float32, dev)
    for name, t in (("D", D), ("dt_bias", dt_bias)):
        if t is not None:
            _expect(name, t, (ch,), torch.float32, dev)
    if z is not None:
        _expect("z", z, x.shape, x.dtype, dev)
    if state is not None:
        _expect("state", state, (b, ch, N), torch.float32, dev)
    _check_starts(starts, b, T, dev)
    _check_state_out(state_out, (b, ch, N), torch.float32, dev, x, dt, A, B, C, D, z, dt_bias, state)
    if state_out is not None and state_out.data_ptr() % 16:
        raise TttError(_lib.TTT_ERR_ALIGN, "state_out is not 16-byte aligned")

    def states(t):
        return t if t.stride(3) == 1 or N == 1 else t.contiguous()
    native = _lib.host().selective(_rows(x), _rows(dt), _aligned(A), states(B), states(C), _dense(D), _rows(z), _dense(dt_bias), _aligned(state),
                                   _dense(starts), softplus, state_out)
    if native is None:
        raise TttError(_lib.TTT_ERR_SHAPE, _lib.last_error() or "unsupported problem for the selective scan")
    return native


def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, activation: Optional[str] = None, eps: float = 1e-5,
               over: str = "token") -> torch.Tensor:
    """Group norm of x [B,T,C] (float32 or bfloat16; any strides that are not negative, with contiguous channels): `groups` groups of
    neighbouring channels, of every token (over="token": nothing reaches from token to token; up to 4096 channels per group) or of every
    sequence with all of its tokens (over="sequence", for layers that see the whole of it).  With u = (x - mean) / sqrt(var + eps) *
    weight + bias (weight, bias [C] of x's type; None: ones, zeros) the result is act(u), or, given a gate [B,T,C], u * act(gate);
    activation None, "silu" or "gelu" (tanh form).  Contiguous [B,T,C].  Differentiable with respect to x, weight, bias and gate, once
    and not in forward mode; statistics and sums are float32, variances are taken from differences."""
    act, place = _NORM_ACTIVATIONS.get(activation), _OVER.get(over)
    if act is None:
        raise _unknown("activation", activation, _NORM_ACTIVATIONS)
    if place is None:
        raise _unknown("over", over, _OVER)
    native = _lib.host().group_norm(x, groups, weight, bias, gate, act, eps, place)
    if native is not None:
        return native
    _check_rows("x", x)
    C = x.shape[2]
    if groups < 1 or C % groups:
        raise TttError(_lib.TTT_ERR_SHAPE, f"channels={C} are not a multiple of groups={groups}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _expect(name, t, (C,), x.dtype, x.device)
    if gate is not None:
        _expect("gate", gate, x.shape, x.dtype, x.device)
    native = _lib.host().group_norm(_rows(x), groups, _dense(weight), _dense(bias), _rows(gate), act, eps, place)
    if native is None:
        raise TttError(_lib.TTT_ERR_SHAPE, _lib.last_error() or "unsupported problem for the group norm")
    return native
