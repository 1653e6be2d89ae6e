"""Training of the outer layer with normed and otherwise rotated queries and keys in front of TTT-Linear and TTT-MLP, against float64
autograd through the same definitions.  Tolerances: float32 those of the layer's other training test (outputs 2e-4, gradients 1e-3);
bfloat16 by norms: forward and backward are six roundings each between the input and a parameter's gradient (projection, heads, inner
loop's operands and result, post norm, output projection), 2^-8 at most of what they round: 12 * 2^-8 < 5e-2."""

import pytest
import torch

from conftest import assert_close
from oracle import rotary_oracle as R
from oracle import ttt_layer_oracle as LO
from oracle import ttt_oracle as O

pytestmark = pytest.mark.gpu


def build(kind, dtype, H=4, F=64, **kw):
    import ttt_rs_b200 as tb
    torch.manual_seed(5)
    cfg = tb.TTTLayerConfig(hidden_size=H * F, num_heads=H, **kw)
    layer = tb.TTT(cfg, device="cuda", dtype=dtype)
    inner = tb.new_inner(cfg, device="cuda", dtype=dtype) if kind == "linear" else \
        tb.FusedTTTMLP(tb.TTTMLP(H, F, cfg.mini_batch_size, 1e-6, device="cuda", dtype=dtype))
    with torch.no_grad():
        for p in [*layer.parameters(), *inner.parameters()]:
            if p.dim() <= 2 and p.shape[-1] != cfg.hidden_size or p.dim() == 1:
                p.add_(torch.randn_like(p) * 0.1)
        layer.learnable_token_idx.mul_(0.1)
    return cfg, layer, inner


def reference(kind, cfg, x, P, I, start):
    """P, I: the layer's and the inner model's parameters by name."""
    B, T, C = x.shape
    H, F = cfg.num_heads, cfg.head_dim
    heads = lambda t: t.reshape(B, T, H, F).transpose(1, 2)  # noqa: E731
    q = x @ P["q_proj"].T
    if cfg.share_qk:
        q, k = (LO.causal_depthwise_conv(q, P[f"{n}_conv_weight"].reshape(C, -1), P[f"{n}_conv_bias"]) for n in "qk")
    else:
        k = x @ P["k_proj"].T
    q, k, v = heads(q), heads(k), heads(x @ P["v_proj"].T)
    if cfg.qk_norm:
        q, k = R.norm(q, P["q_norm_weight"]), R.norm(k, P["k_norm_weight"])
    rc = cfg.rotary_config()
    if rc is not None:
        q, k = (R.rotate(t, rc, torch.arange(start, start + T)) for t in (q, k))
    lr = cfg.base_lr / F * torch.sigmoid(torch.einsum("btc,hc->bht", x, P["learnable_ttt_lr_weight"][..., 0]) + P["learnable_ttt_lr_bias"][None])
    te = torch.clamp_min(1.0 / torch.arange(1, cfg.mini_batch_size + 1).double() + P["learnable_token_idx"], 0.0).repeat(T // cfg.mini_batch_size)
    first = lambda n: I[n][None].expand(B, *I[n].shape)  # noqa: E731
    states = [first(n) for n in (("weight_init", "bias_init") if kind == "linear" else ("w1_init", "b1_init", "w2_init", "b2_init"))]
    scan = O.ttt_linear_forward if kind == "linear" else O.ttt_mlp_forward
    out = scan(q, k, v, *states, te, lr, I["ln_weight"], I["ln_bias"], mini_batch=cfg.mini_batch_size, eps=1e-6)["output"]
    return LO.layer_epilogue(out, x, P, use_gate=cfg.use_gate) @ P["o_proj"].T


CONFIGS = [dict(qk_norm=True), dict(qk_norm=True, rope_layout="half", rotary_dim=32, pos_encoding="rope_global", use_gate=True),
           dict(rope_scaling="linear", rope_factor=4.0), dict(qk_norm=True, share_qk=True, pos_encoding="none")]


@pytest.mark.parametrize("kw", CONFIGS)
@pytest.mark.parametrize("kind,dtype", [("linear", torch.float32), ("linear", torch.bfloat16), ("mlp", torch.bfloat16)])
def test_training(kind, dtype, kw):
    import ttt_rs_b200 as tb
    cfg, layer, inner = build(kind, dtype, **kw)
    B, T, start = 2, 64, 16
    x, gy = (torch.randn(B, T, cfg.hidden_size) * s for s in (0.5, 1.0))
    x, gy = x.to(dtype), gy.to(dtype)
    P = {n: p.detach().double().cpu().requires_grad_() for n, p in layer.named_parameters()}
    I = {n: p.detach().double().cpu().requires_grad_() for n, p in inner.inner.named_parameters()}
    xr, xg = x.double().requires_grad_(), x.cuda().requires_grad_()
    want = reference(kind, cfg, xr, P, I, start)
    want.backward(gy.double())
    y = layer(xg, inner, inner.init_state(B), start_idx=start)
    y.backward(gy.cuda())
    tb.check_status()
    pairs = [("output", y, want, 2e-4), ("input", xg.grad, xr.grad, 1e-3)]
    pairs += [(n, p.grad, P[n].grad, 1e-3) for n, p in layer.named_parameters()]
    pairs += [(n, p.grad, I[n].grad, 1e-3) for n, p in inner.inner.named_parameters()]
    for name, a, b, tol in pairs:
        assert a is not None, name
        if dtype == torch.float32:
            assert_close(a.reshape(b.shape), b, tol, f"own heads, {kind}: {name}")
        else:
            e = ((a.detach().double().cpu().reshape(b.shape) - b).norm() / b.norm()).item()
            assert e <= 5e-2, (name, e)


def test_captured_tokens_of_the_recurrence():
    """A token's step in a graph: the new state copied to where the captured one is read, between replays."""
    import ttt_rs_b200 as tb
    cfg = tb.TTTLayerConfig(hidden_size=256, num_heads=4, qk_norm=True, pos_encoding="none")
    layer, inner = tb.TTT(cfg, device="cuda", dtype=torch.bfloat16), tb.new_gated_inner(cfg, device="cuda")
    x = torch.randn(3, 12, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        eager = inner.init_state(3)
        want = [layer(x[:, t:t + 1].contiguous(), inner, eager) for t in range(12)]
        state, token = inner.init_state(3), x[:, :1].clone()
        held, graph = state.weight, torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = layer(token, inner, state)
        for t in range(12):
            token.copy_(x[:, t:t + 1])
            graph.replay()
            assert torch.equal(out, want[t])
            held.copy_(state.weight)
    assert torch.equal(held, eager.weight)
