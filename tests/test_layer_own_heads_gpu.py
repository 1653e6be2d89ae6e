"""The outer layer with normed and otherwise rotated queries and keys, and with the gated linear recurrence as its inner model:
projections, norm and rotation, recurrence, post norm and output projection as they run together, against a float64 composition of
the same definitions.  Tolerances: those of the layer's other tests (5e-4 float32 with its gradients, 5e-2 of rows and
gradients in bfloat16, where every step between two kernels is a rounding of its own)."""

import math

import pytest
import torch

from conftest import assert_close
from oracle import gated_oracle as G
from oracle import rotary_oracle as R

pytestmark = pytest.mark.gpu


def build(dtype, H=4, F=64, seed=0, **kw):
    import ttt_rs_b200 as tb
    torch.manual_seed(seed)
    cfg = tb.TTTLayerConfig(hidden_size=H * F, num_heads=H, **kw)
    layer = tb.TTT(cfg, device="cuda", dtype=dtype)
    with torch.no_grad():
        for p in layer.parameters():
            if p.dim() == 1:
                p.add_(torch.randn_like(p) * 0.1)
    inner = tb.new_gated_inner(cfg, device="cuda")
    return cfg, layer, inner


def reference(x, layer, inner, cfg, w, start=0):
    """The layer's definition in float64 on the CPU, differentiable with respect to x, the parameters P and w."""
    import ttt_rs_b200 as tb  # noqa: F401
    P = {k: v.detach().double().cpu().requires_grad_() for k, v in layer.named_parameters()}
    D = {k: v.detach().double().cpu().requires_grad_() for k, v in inner.inner.named_parameters()}
    B, T, C = x.shape
    H, F = cfg.num_heads, cfg.head_dim
    heads = lambda t: t.reshape(B, T, H, F).transpose(1, 2)  # noqa: E731
    q, v = x @ P["q_proj"].T, heads(x @ P["v_proj"].T)
    if cfg.share_qk:
        def conv(t, weight, bias):
            pad = torch.nn.functional.pad(t.transpose(1, 2), (weight.shape[-1] - 1, 0))
            return torch.nn.functional.conv1d(pad, weight, bias, groups=C).transpose(1, 2)
        q, k = conv(q, P["q_conv_weight"], P["q_conv_bias"]), conv(q, P["k_conv_weight"], P["k_conv_bias"])
    else:
        k = x @ P["k_proj"].T
    q, k = heads(q), heads(k)
    if cfg.qk_norm:
        q, k = R.norm(q, P["q_norm_weight"]), R.norm(k, P["k_norm_weight"])
    rc = cfg.rotary_config()
    if rc is not None:
        pos = torch.arange(start, start + T)
        q, k = R.rotate(q, rc, pos), R.rotate(k, rc, pos)
    z = torch.einsum("btc,hc->bht", x, P["learnable_ttt_lr_weight"][..., 0]) + P["learnable_ttt_lr_bias"][None]
    beta = cfg.base_lr / F * torch.sigmoid(z)
    g = torch.log1p(-torch.sigmoid(D["decay_logit"])[:, None] * torch.sigmoid(z))
    o, w = G.gated_forward(q, k, v, g, beta, w)
    y = o.transpose(1, 2).reshape(B, T, C)
    y = torch.nn.functional.layer_norm(y, (C,), P["post_norm_weight"], P["post_norm_bias"], 1e-6)
    if cfg.use_gate:
        y = y * torch.nn.functional.gelu(x @ P["g_proj"].T, approximate="tanh")
    return y @ P["o_proj"].T, w, P, D


CONFIGS = [dict(qk_norm=True), dict(qk_norm=True, rope_layout="half", rotary_dim=32, pos_encoding="rope_global", use_gate=True),
           dict(rope_layout="half"), dict(qk_norm=True, pos_encoding="none"), dict(qk_norm=True, share_qk=True),
           dict(rope_scaling="by_parts", rope_factor=8.0, rope_original_length=64, pos_encoding="rope_global"), dict()]


@pytest.mark.parametrize("kw", CONFIGS)
@pytest.mark.parametrize("T", [1, 70])
def test_layer_forward_float32(kw, T):
    cfg, layer, inner = build(torch.float32, **kw)
    x = torch.randn(2, T, 256) * 0.5
    state = inner.init_state(2)
    w0 = state.weight.double().cpu()
    want, w, _, _ = reference(x.double(), layer, inner, cfg, w0, start=3)
    with torch.no_grad():
        y = layer(x.cuda(), inner, state, start_idx=3)
    assert_close(y, want, 5e-4, "own heads: layer output")
    assert_close(state.weight, w, 5e-4, "own heads: state")


@pytest.mark.parametrize("kw", CONFIGS)
def test_layer_gradients_float32(kw):
    cfg, layer, inner = build(torch.float32, **kw)
    x, u = torch.randn(2, 90, 256) * 0.5, torch.randn(2, 90, 256)
    xd = x.double().requires_grad_()
    dev = x.cuda().requires_grad_()
    state = inner.init_state(2)
    want, _, P, D = reference(xd, layer, inner, cfg, state.weight.double().cpu())
    (want * u.double()).sum().backward()
    y = layer(dev, inner, state)
    (y * u.cuda()).sum().backward()
    assert_close(y, want.detach(), 5e-4, "own heads: layer output")
    assert_close(dev.grad, xd.grad, 5e-4, "own heads: d x")
    used = {k: v for k, v in layer.named_parameters() if k != "learnable_token_idx"}  # (every token is an update of its own)
    for name, p in used.items():
        assert_close(p.grad, P[name].grad, 5e-4, f"own heads: d {name}")
    assert_close(inner.inner.decay_logit.grad, D["decay_logit"].grad, 5e-4, "own heads: d decay_logit")


def test_layer_bfloat16_and_token_by_token():
    """A prompt and then single tokens, positions going on, against the whole sequence at once."""
    cfg, layer, inner = build(torch.bfloat16, qk_norm=True, rope_layout="half", pos_encoding="rope_global", use_gate=True)
    x = (torch.randn(3, 40, 256) * 0.5).bfloat16()
    state = inner.init_state(3)
    want, _, _, _ = reference(x.double(), layer, inner, cfg, state.weight.double().cpu())
    with torch.no_grad():
        whole = layer(x.cuda(), inner, inner.init_state(3))
        state = inner.init_state(3)
        parts = [layer(x[:, :33].cuda(), inner, state)]
        for t in range(33, 40):
            parts.append(layer(x[:, t:t + 1].cuda(), inner, state, start_idx=t))
    assert_close(whole, want, 5e-2, "own heads: bf16 layer output")
    assert_close(torch.cat(parts, 1), want, 5e-2, "own heads: bf16 token by token")


def test_training_steps_in_bfloat16_run():
    cfg, layer, inner = build(torch.bfloat16, qk_norm=True, rope_layout="half")
    params = list(layer.parameters()) + list(inner.parameters())
    opt = torch.optim.SGD(params, lr=1e-3)
    x = torch.randn(2, 130, 256, device="cuda", dtype=torch.bfloat16)
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        y = layer(x, inner, inner.init_state(2))
        y.float().square().mean().backward()
        assert all(torch.isfinite(p.grad).all() for p in params if p.grad is not None)
        assert layer.q_norm_weight.grad.abs().sum() > 0 and inner.inner.weight_init.grad.abs().sum() > 0
        opt.step()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ttt_linear_behind_normed_heads(dtype):
    """The same heads in front of the TTT-Linear inner model, its decode graphs included."""
    import ttt_rs_b200 as tb
    from oracle import ttt_oracle as O
    cfg, layer, _ = build(dtype, qk_norm=True, rope_layout="half")
    inner = tb.new_inner(cfg, device="cuda", dtype=dtype, allow_partial=True, partial_in_place=True)
    x = (torch.randn(2, 32, 256) * 0.5).to(dtype).cuda()
    with torch.no_grad():
        inputs, _, _ = layer.get_inner_loop_inputs(x, 0)
        y = layer(x, inner, inner.init_state(2))
        st = inner.init_state(2)
        want = O.ttt_linear_forward(*[t.double().cpu() for t in (
            inputs.qkv.xq, inputs.qkv.xk, inputs.qkv.xv, st.weight, st.bias, inputs.token_eta, inputs.ttt_lr_eta,
            inner.inner.ln_weight, inner.inner.ln_bias)], mini_batch=16)["output"]
        z = torch.nn.functional.layer_norm(want.transpose(1, 2).reshape(2, 32, 256), (256,), layer.post_norm_weight.double().cpu(),
                                           layer.post_norm_bias.double().cpu(), 1e-6) @ layer.o_proj.double().cpu().T
        assert_close(y, z, 5e-2 if dtype == torch.bfloat16 else 5e-4, "normed heads, TTT-Linear")
        one, many = inner.init_state(2), inner.init_state(2)
        graphs = tb.DecodeGraphs(layer, inner, many, 2)
        for t in range(20):
            a, b = layer(x[:, t:t + 1], inner, one, t % 16), graphs.step(x[:, t:t + 1], t)
            if dtype == torch.bfloat16:
                assert torch.equal(a, b)
            else:
                # float32 projections are library products, which may sum their 256 terms in another order when captured: 256 * 2^-24
                # of the terms' size per product, three products and twenty steps of state behind one another below 1e-3; measured 1e-6
                assert_close(b, a, 5e-4, "normed heads, captured steps")
    with pytest.raises(ValueError):
        tb.DecodeGraphs(layer, tb.new_gated_inner(cfg, device="cuda"), None, 2)


def test_layer_on_its_own_stream_and_in_a_graph():
    cfg, layer, inner = build(torch.bfloat16, qk_norm=True)
    x = torch.randn(2, 700, 256, device="cuda", dtype=torch.bfloat16)
    state = inner.init_state(2)
    w0 = state.weight.clone()
    with torch.no_grad():
        want = layer(x, inner, state)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            state.weight = w0.clone()
            got = layer(x, inner, state)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        state.weight = w0
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = layer(x, inner, state)
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_refused_configurations():
    import ttt_rs_b200 as tb
    for kw in (dict(rope_layout="other"), dict(rotary_dim=65), dict(rope_scaling="by_parts", rope_factor=2.0)):
        with pytest.raises(ValueError):
            tb.TTT(tb.TTTLayerConfig(hidden_size=128, num_heads=2, **kw), device="cuda")
    assert math.isclose(tb.TTTLayerConfig(128, 2, rope_scaling="by_parts", rope_factor=math.e, rope_original_length=64).rotary_config().size, 1.1)


def test_base_lr_of_the_recurrence_is_positive():
    import ttt_rs_b200 as tb
    with pytest.raises(ValueError):
        tb.GatedLinear(2, 64, base_lr=0.0)
