"""Gated linear recurrence as an inner model beside TTT-Linear and TTT-MLP (csrc/ttt_gated_*.cu):

    W_t = exp(g_t) W_{t-1} + beta_t k_t^T v_t,      o_t = q_t W_t

for every (batch, head) stream, W [F, F] in float32.  It is what the TTT inner loop becomes when the reconstruction loss is
replaced by -<k W, v> with weight decay: the update is then linear in W, needs no mini-batches, and a sequence can be scanned
in chunks.  (The reference has no such inner model.)
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import TttError
from .fused import TTTInputsInner, _expect, _per_sequence, device_status


def _strided(t: torch.Tensor) -> torch.Tensor:
    """t [B,H,T,F] as the kernels take it: rows contiguous and, like the base, on 16 bytes; a copy where it is not."""
    es = t.element_size()
    ok = t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(
        n == 1 or (s > 0 and s * es % 16 == 0) for n, s in zip(t.shape[:3], t.stride()[:3]))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def fused_gated_linear(xq: torch.Tensor, xk: torch.Tensor, xv: torch.Tensor, log_decay: torch.Tensor,
                       beta: Optional[torch.Tensor] = None,
                       weight: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(output [B,H,T,F], state behind the last token [B,H,F,F] float32) of the recurrence over xq, xk, xv [B,H,T,F] (float32 or
    bfloat16, head_dim 64 or 32; views of [B,T,H,F] or of a projection are read where they lie), from the state `weight`
    [B,H,F,F] float32 (None: zeros).  log_decay [B,H,T] float32, at most 0; -inf forgets everything before the token, so that
    sequences may follow one another in one row.  beta [B,H,T] float32 (None: ones).  Differentiable with respect to all six,
    through both results (once: gradients of gradients are refused); without gradients a call of up to 16 tokens runs as a decode
    step.  Derivatives in forward mode are refused.  A NaN or an infinity in a token reaches results of the 64 tokens around it, and no
    reset forgets one in the state.

    The state, log_decay, beta, weight and their gradients are float32 throughout (4e-7 of their norm, from bfloat16 inputs too), and so are all
    results of float32 inputs (1e-7).  bfloat16 results are rounded more than once, each time by 2^-8 at most: the decayed products of
    queries and keys (of output gradients and values) and the state (its gradient) become bfloat16 operands.  output, grad_xq, grad_xk and
    grad_xv are off by 2.3e-3 to 2.4e-3 of their norm, where one rounding of exact results leaves 1.7e-3.  (float32 inputs take three to
    four times as long.)"""
    native = _lib.host().gated(xq, xk, xv, log_decay, beta, weight)
    if native is not None:
        return native
    if not xq.is_cuda:
        raise TttError(_lib.TTT_ERR_CUDA, "inputs must be CUDA tensors: this operator has no CPU path")
    if xq.dim() != 4:
        raise TttError(_lib.TTT_ERR_SHAPE, f"xq must be [batch, heads, seq_len, head_dim], got {tuple(xq.shape)}")
    if xq.dtype not in (torch.float32, torch.bfloat16):
        raise TttError(_lib.TTT_ERR_UNSUPPORTED, f"unsupported dtype {xq.dtype}")
    B, H, T, F = xq.shape
    dev = xq.device
    if min(B, H, T) == 0:
        raise TttError(_lib.TTT_ERR_SHAPE, "batch, heads and seq_len must be positive")
    if F not in (32, 64):
        raise TttError(_lib.TTT_ERR_UNSUPPORTED, f"Unsupported head_dim={F} (supported: 64, 32)")
    for name, t in (("xk", xk), ("xv", xv)):
        _expect(name, t, (B, H, T, F), xq.dtype, dev)
    _expect("log_decay", log_decay, (B, H, T), torch.float32, dev)
    if beta is not None:
        _expect("beta", beta, (B, H, T), torch.float32, dev)
    if weight is not None:
        _expect("weight", weight, (B, H, F, F), torch.float32, dev)
    device_status(dev)
    native = _lib.host().gated(_strided(xq), _strided(xk), _strided(xv), log_decay.contiguous(),
                               None if beta is None else beta.contiguous(), None if weight is None else _aligned(weight))
    if native is None:
        raise TttError(_lib.TTT_ERR_SHAPE, _lib.last_error() or "unsupported problem for the gated linear recurrence")
    return native


@dataclass
class GatedLinearState:
    weight: torch.Tensor  # [batch, heads, F, F] float32


class GatedLinear(torch.nn.Module):
    """Parameter holder: weight_init [H,F,F] float32 ~ N(0, 0.02) and, per head, the logit of the weight decay (of another type after
    `.to(dtype)` of a whole model; states and gates are float32 all the same).  With the
    layer's learning rate eta_t = base_lr sigmoid(.) / F of a token, head h writes with beta_t = eta_t and keeps
    1 - sigmoid(decay_logit_h) sigmoid(.) of its state; the heads' strongest decays start spread from 2^-1 to 2^-7."""

    def __init__(self, num_heads: int, head_dim: int, base_lr: float = 1.0, device=None):
        super().__init__()
        if not base_lr > 0.0:
            raise ValueError(f"base_lr must be positive (got {base_lr})")
        self.num_heads, self.head_dim, self.base_lr = num_heads, head_dim, base_lr
        kw = dict(device=device, dtype=torch.float32)
        self.weight_init = torch.nn.Parameter(torch.randn(num_heads, head_dim, head_dim, **kw) * 0.02)
        most = 2.0 ** -(1 + 6 * torch.arange(num_heads, **kw) / num_heads)
        self.decay_logit = torch.nn.Parameter(torch.log(most) - torch.log1p(-most))

    def init_state(self, batch_size: int) -> GatedLinearState:
        return GatedLinearState(_per_sequence(self.weight_init.float(), batch_size))

    def gates(self, ttt_lr_eta: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """(log_decay, beta) [B,H,T] float32 from the layer's learning rates."""
        beta = ttt_lr_eta.float()
        forget = torch.sigmoid(self.decay_logit.float())[:, None] * (beta * (self.head_dim / self.base_lr))
        return torch.log1p(-forget.clamp(max=1.0 - 2.0 ** -20)), beta


class FusedGatedLinear(torch.nn.Module):
    """The recurrence with the `forward(state, inputs)` interface of the inner models, for `TTT` and for callers of their own:
    any sequence length, single tokens included, and the state advanced from call to call: `state.weight` is another tensor behind every
    call.  (A captured call reads the state where it lay at the capture: keep that tensor, and copy the new state into it between
    replays.)  token_eta is not used: every token is an update of its own."""

    def __init__(self, inner: GatedLinear):
        super().__init__()
        self.inner = inner

    @staticmethod
    def name() -> str:
        return "FusedGatedLinear"

    def init_state(self, batch_size: int) -> GatedLinearState:
        return self.inner.init_state(batch_size)

    def forward(self, state: GatedLinearState, inputs: TTTInputsInner) -> torch.Tensor:
        log_decay, beta = self.inner.gates(inputs.ttt_lr_eta)
        q = inputs.qkv
        out, state.weight = fused_gated_linear(q.xq, q.xk, q.xv, log_decay, beta, state.weight)
        return out
