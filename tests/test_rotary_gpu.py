"""Rotary positions, and the norm of queries and keys with them, against the float64 oracle.

Bounds.  `mag` of a rotated feature is |a| + |b| of its pair times the size.  float32: the sine and cosine are off by 2^-22 at
most (an angle of half a turn held in 24 bits, and their own error), the two products and their sum by three roundings:
2^-21 mag.  The norm adds a sum of F squares (F 2^-24 in the worst order), a reciprocal root and two products: (F + 8) 2^-24.
Gradients add a second sum of F products: 2 (F + 8) 2^-24 of what its terms amount to.  bf16 results: one rounding, 2^-8 of the
result.  Gradients of the weights: float32 sums over the rows, a few hundred of them in one register: 2^-14 of the terms'
absolute sum at most, and the result's rounding."""

import math

import pytest
import torch

from oracle import rotary_oracle as O

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def within(got, want, tol, name):
    got = got.detach().double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    over = (got - want).abs() - tol - 2 ** -126
    assert over.max() <= 0, f"{name}: off by {(got - want).abs().max():.3g}, {over.max():.3g} over the bound"


def pair_mag(x, cfg):
    """|a| + |b| of every feature's pair (|x| where it has none)."""
    r = cfg.rotary_dim or cfg.head_dim
    y = x.abs().clone()
    if cfg.layout == "half":
        s = y[..., :r // 2] + y[..., r // 2:r]
        y[..., :r // 2] = y[..., r // 2:r] = s
    else:
        s = y[..., 0:r:2] + y[..., 1:r:2]
        y[..., 0:r:2] = y[..., 1:r:2] = s
    return y


def values(B, H, T, F, dtype, seed=0, layout="heads"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, T, F, generator=g).to(dtype)
    if layout == "heads":
        d = x.cuda()
    elif layout == "tokens":
        d = x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    elif layout == "columns":
        d = torch.full((B, T, H * F + 24), math.nan, dtype=dtype, device="cuda")[..., 8:8 + H * F].unflatten(-1, (H, F)).transpose(1, 2)
        d.copy_(x)
    else:  # rows that start anywhere
        d = torch.full((B, H, T, F + 3), math.nan, dtype=dtype, device="cuda")[..., 1:F + 1]
        d.copy_(x)
    return x.double(), d


def check_rotary(cfg, B, H, T, dtype, layout="heads", start=0, positions=None, seed=0):
    import ttt_rs_b200 as tb
    rot = tb.Rotary(cfg, device="cuda")
    x, d = values(B, H, T, cfg.head_dim, dtype, seed, layout)
    pos = torch.arange(start, start + T) if positions is None else positions
    want, size = O.rotate(x, cfg, pos), cfg.size
    mag = pair_mag(x, cfg) * size
    tol = 2 ** -21 * mag + HALF_STEP[dtype] * want.abs()
    p = None if positions is None else positions.cuda()
    with torch.no_grad():
        y = tb.rotary(d, rot, start_idx=start, positions=p)
    assert y.is_contiguous()
    within(y, want, tol, "rotated")
    # back again: the gradient is the rotation by the negative angles
    u = torch.randn(B, H, T, cfg.head_dim, generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
    leaf = d.detach().requires_grad_()
    (dx,) = torch.autograd.grad(tb.rotary(leaf, rot, start_idx=start, positions=p), leaf, u.cuda())
    xr = x.clone().requires_grad_()
    (want_dx,) = torch.autograd.grad(O.rotate(xr, cfg, pos), xr, u.double())
    within(dx, want_dx, 2 ** -21 * pair_mag(u.double(), cfg) * size + HALF_STEP[dtype] * want_dx.abs(), "gradient")
    return rot, d, y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pairs", ["interleaved", "half"])
@pytest.mark.parametrize("F,rdim", [(64, None), (64, 16), (64, 20), (128, 64), (80, 24), (256, None), (34, None), (2, None), (32, 8)])
def test_rotary_shapes(F, rdim, pairs, dtype):
    import ttt_rs_b200 as tb
    cfg = tb.RotaryConfig(head_dim=F, rotary_dim=rdim, layout=pairs)
    check_rotary(cfg, 2, 3, 37, dtype, start=5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["tokens", "columns", "odd"])
@pytest.mark.parametrize("pairs", ["interleaved", "half"])
def test_rotary_layouts(layout, pairs, dtype):
    import ttt_rs_b200 as tb
    check_rotary(tb.RotaryConfig(head_dim=64, layout=pairs), 2, 5, 33, dtype, layout=layout)


@pytest.mark.parametrize("T,B,H", [(1, 1, 1), (1, 8, 12), (2, 3, 1), (1000, 1, 7), (129, 2, 40)])
def test_rotary_sizes(T, B, H):
    import ttt_rs_b200 as tb
    check_rotary(tb.RotaryConfig(head_dim=64), B, H, T, torch.bfloat16, start=100)


@pytest.mark.parametrize("pairs", ["interleaved", "half"])
@pytest.mark.parametrize("scaling", [dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
                                     dict(scaling="by_parts", factor=32.0, original_length=4096), dict(wrap=16), dict(theta=1.0)])
def test_far_positions_keep_their_angles(scaling, pairs):
    """Angles at a million and more: a float32 product of position and frequency would be off by 0.03 and more."""
    import ttt_rs_b200 as tb
    cfg = tb.RotaryConfig(head_dim=64, layout=pairs, **scaling)
    for start in (0, (1 << 20) - 3, (1 << 31) + 11):
        check_rotary(cfg, 1, 2, 9, torch.float32, start=start)


def test_given_positions():
    import ttt_rs_b200 as tb
    g = torch.Generator().manual_seed(2)
    for shape, dtype in (((50,), torch.int64), ((3, 50), torch.int64), ((3, 50), torch.int32)):
        pos = torch.randint(-70000, 70000, shape, generator=g, dtype=dtype)
        check_rotary(tb.RotaryConfig(head_dim=64), 3, 2, 50, torch.float32, positions=pos)
        check_rotary(tb.RotaryConfig(head_dim=64, wrap=16), 3, 2, 50, torch.bfloat16, positions=pos)


def test_in_place_and_into_given_results():
    import ttt_rs_b200 as tb
    for pairs in ("interleaved", "half"):
        rot = tb.Rotary(tb.RotaryConfig(head_dim=64, layout=pairs), device="cuda")
        _, d = values(2, 3, 40, 64, torch.bfloat16, layout="columns")
        with torch.no_grad():
            y = tb.rotary(d, rot)
            other = torch.empty(2, 40, 3, 64, dtype=d.dtype, device="cuda").transpose(1, 2)
            assert tb.rotary(d, rot, out=other) is not None and torch.equal(other, y)
            tb.rotary(d, rot, out=d)
        assert torch.equal(d, y)


def test_the_layers_own_rotation_is_one_of_these():
    """Neighbouring pairs over the whole head, positions modulo the mini-batch: what ttt_layer_prologue does."""
    import ttt_rs_b200 as tb
    cfg = tb.TTTLayerConfig(hidden_size=128, num_heads=2)
    proj = torch.randn(2, 48, 3 * 128 + 8, device="cuda")
    xq, xk, _, _ = tb.layer_prologue(proj, cfg, q_col=0, k_col=128, v_col=256, lr_col=384, lr_bias=None, start_idx=3)
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64, wrap=16), device="cuda")
    for x, col in ((xq, 0), (xk, 128)):
        y = tb.rotary(proj[..., col:col + 128].unflatten(-1, (2, 64)).transpose(1, 2), rot, start_idx=3)
        assert (y - x).abs().max() < 1e-5


# ---- norm and rotation -------------------------------------------------------------------------------------------------

def check_qk(cfg, B, H, Hk, T, F, dtype, layout="heads", weights=(True, True), start=0, scale=1.0, eps=1e-6):
    import ttt_rs_b200 as tb
    rot = None if cfg is None else tb.Rotary(cfg, device="cuda")
    size = 1.0 if cfg is None else cfg.size
    some = cfg or tb.RotaryConfig(head_dim=F)
    pos = torch.arange(start, start + T)
    turn = (lambda x: x) if cfg is None else (lambda x: O.rotate(x, cfg, pos))
    mags = (lambda x: x.abs()) if cfg is None else (lambda x: pair_mag(x, some) * size)
    g = torch.Generator().manual_seed(11)
    xs, ws, us = [], [], []
    for n, heads in enumerate((H, Hk)):
        x, d = values(B, heads, T, F, dtype, seed=n, layout=layout)
        d.mul_(scale)
        xs.append((d.double().cpu(), d.detach().requires_grad_()))
        w = (1 + 0.2 * torch.randn(F, generator=g)).to(dtype) if weights[n] else None
        ws.append((None if w is None else w.double(), None if w is None else w.cuda().requires_grad_()))
        us.append(torch.randn(B, heads, T, F, generator=g).to(dtype))
    ys = tb.qk_norm_rotary(xs[0][1], xs[1][1], ws[0][1], ws[1][1], rot, eps=eps, start_idx=start)
    with torch.no_grad():
        zs = tb.qk_norm_rotary(xs[0][1], xs[1][1], ws[0][1], ws[1][1], rot, eps=eps, start_idx=start)
    assert all(torch.equal(a, b) for a, b in zip(ys, zs))
    leaves = [x[1] for x in xs] + [w[1] for w in ws if w[1] is not None]
    grads = torch.autograd.grad(ys, leaves, [u.cuda() for u in us])
    dws = iter(grads[2:])
    half = HALF_STEP[dtype]
    for n in range(2):
        x, w, u = xs[n][0].clone().requires_grad_(), ws[n][0], us[n].double()
        if w is not None:
            w = w.clone().requires_grad_()
        want = turn(O.norm(x, w, eps))
        got = torch.autograd.grad(want, [x] if w is None else [x, w], u)
        want = want.detach()
        e = (F + 16) * 2 ** -24
        within(ys[n], want, (2 ** -21 + e) * mags(O.norm(x, w, eps).detach()) + half * want.abs(), f"result {n}")
        x, wv = x.detach(), 1.0 if w is None else w.detach()
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        ur = mags(u)  # (the rotation back)
        mag = r * ur * abs(wv) + x.abs() * r ** 3 * (ur * abs(wv) * x.abs()).mean(-1, keepdim=True)
        within(grads[n], got[0], (2 ** -20 + 4 * e) * mag + half * got[0].abs(), f"gradient {n}")
        if w is not None:
            m = (ur * x.abs() * r).sum((0, 1, 2))
            within(next(dws), got[1], 2 ** -14 * m + half * got[1].abs(), f"weight's gradient {n}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pairs", ["interleaved", "half"])
@pytest.mark.parametrize("F,rdim", [(64, None), (128, 32), (96, 20), (256, None), (34, None), (32, 8)])
def test_qk_shapes(F, rdim, pairs, dtype):
    import ttt_rs_b200 as tb
    check_qk(tb.RotaryConfig(head_dim=F, rotary_dim=rdim, layout=pairs), 2, 6, 3, 37, F, dtype, start=1000)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["tokens", "columns", "odd"])
def test_qk_layouts(layout, dtype):
    import ttt_rs_b200 as tb
    check_qk(tb.RotaryConfig(head_dim=64, layout="half"), 2, 5, 5, 50, 64, dtype, layout=layout)


@pytest.mark.parametrize("B,H,Hk,T", [(1, 1, 1, 1), (8, 12, 4, 1), (1, 32, 1, 300), (4, 3, 12, 513)])
def test_qk_sizes(B, H, Hk, T):
    import ttt_rs_b200 as tb
    check_qk(tb.RotaryConfig(head_dim=64), B, H, Hk, T, 64, torch.bfloat16)


@pytest.mark.parametrize("weights", [(True, False), (False, True), (False, False)])
def test_qk_without_weights_or_rotation(weights):
    import ttt_rs_b200 as tb
    check_qk(tb.RotaryConfig(head_dim=64), 2, 3, 2, 20, 64, torch.float32, weights=weights)
    check_qk(None, 2, 3, 2, 20, 64, torch.bfloat16, weights=weights)


@pytest.mark.parametrize("scale", [1e-12, 1e-4, 1e4])
def test_qk_small_and_large_rows(scale):
    """Rows far below and far above sqrt(eps)."""
    import ttt_rs_b200 as tb
    check_qk(tb.RotaryConfig(head_dim=64), 1, 2, 2, 9, 64, torch.float32, scale=scale)


def test_qk_zero_rows():
    import ttt_rs_b200 as tb
    q = torch.zeros(1, 2, 5, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, _ = tb.qk_norm_rotary(q, q, w, w, tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda"))
    assert (y == 0).all()
    dq, dw = torch.autograd.grad(y.sum(), [q, w])
    assert torch.isfinite(dq).all() and (dw == 0).all()


def test_the_same_twice_and_replayed_from_a_graph():
    import ttt_rs_b200 as tb
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64, layout="half"), device="cuda")
    _, q = values(3, 4, 700, 64, torch.bfloat16, layout="tokens")
    _, k = values(3, 2, 700, 64, torch.bfloat16, seed=1, layout="tokens")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)

    def step():
        ql, kl = q.detach().requires_grad_(), k.detach().requires_grad_()
        ys = tb.qk_norm_rotary(ql, kl, w, w, rot)
        grads = torch.autograd.grad(ys, [ql, kl, w], [torch.ones_like(y) for y in ys])
        return [y.detach() for y in ys] + list(grads)  # (no eager graph of w may live while its backward is captured)

    a, b = step(), step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, c))


def test_refusals():
    import ttt_rs_b200 as tb
    from ttt_rs_b200 import _lib as L
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda")
    x = torch.zeros(2, 3, 8, 64, device="cuda")

    def refused(code, call):
        with pytest.raises(tb.TttError) as e:
            call()
        assert e.value.code == code

    refused(L.TTT_ERR_CUDA, lambda: tb.rotary(x.cpu(), rot))
    refused(L.TTT_ERR_UNSUPPORTED, lambda: tb.rotary(x.half(), rot))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(x[..., :32], rot))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(x[0], rot))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(x[:, :, :0], rot))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(x, rot, positions=torch.zeros(9, dtype=torch.int64, device="cuda")))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(x, rot, positions=torch.zeros(8, device="cuda")))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(x, rot, positions=torch.zeros(8, dtype=torch.int64)))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(x, rot, out=torch.zeros(2, 3, 8, 64, dtype=torch.bfloat16, device="cuda")))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(x, rot, out=x[:, :, :1].expand(2, 3, 8, 64)))
    refused(L.TTT_ERR_SHAPE, lambda: tb.rotary(x, tb.Rotary(tb.RotaryConfig(head_dim=64), device="cpu")))
    refused(L.TTT_ERR_UNSUPPORTED, lambda: tb.rotary(x.clone().requires_grad_(), rot, out=x))
    refused(L.TTT_ERR_SHAPE, lambda: tb.qk_norm_rotary(x, x[:, :, :4], rot=rot))
    refused(L.TTT_ERR_SHAPE, lambda: tb.qk_norm_rotary(x, x, torch.ones(64, device="cuda", dtype=torch.bfloat16), rot=rot))
    refused(L.TTT_ERR_SHAPE, lambda: tb.qk_norm_rotary(x, x, eps=-1.0))


def test_results_that_lie_over_another_tensor_are_refused():
    import ttt_rs_b200 as tb
    from ttt_rs_b200 import _lib as L
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda")
    flat = torch.zeros(2 * 3 * 8 * 64 + 64, device="cuda")
    x, moved = flat[:-64].view(2, 3, 8, 64), flat[64:].view(2, 3, 8, 64)
    q, k = torch.zeros(2, 2, 3, 8, 64, device="cuda")

    def refused(call):
        with pytest.raises(tb.TttError) as e:
            call()
        assert e.value.code == L.TTT_ERR_SHAPE

    refused(lambda: tb.rotary(x, rot, out=moved))
    refused(lambda: tb.rotary(x, rot, out=flat.as_strided((2, 3, 8, 64), (3 * 64, 64, 64, 1))))
    refused(lambda: tb.qk_norm_rotary(q, k, rot=rot, out=(k, q)))
    refused(lambda: tb.qk_norm_rotary(q, k, rot=rot, out=(q, q)))
    refused(lambda: tb.qk_norm_rotary(x, k, rot=rot, out=(moved, k)))
    both = torch.zeros(2, 8, 2, 3, 64, device="cuda")  # columns of one projection, each normed where it lies
    cols = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    got = tb.qk_norm_rotary(*cols, rot=rot, out=cols)
    assert got[0].data_ptr() == cols[0].data_ptr()


def test_gradients_of_gradients_are_refused():
    import ttt_rs_b200 as tb
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda")
    x, w = torch.randn(2, 3, 8, 64, device="cuda").requires_grad_(), torch.ones(64, device="cuda").requires_grad_()
    for y in (tb.rotary(x, rot), tb.qk_norm_rotary(x, x, w, w, rot)[0]):
        (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="not differentiable"):
            dx.sum().backward()


def test_rotary_offsets_behind_32_bits():
    import ttt_rs_b200 as tb
    rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cuda")
    B, T, H, F = 9, 1 << 20, 4, 64
    x = torch.zeros(B, T, H, F, device="cuda", dtype=torch.bfloat16)
    x[-1, -5:] = torch.randn(5, H, F, device="cuda")
    y = tb.rotary(x.transpose(1, 2), rot)
    want = tb.rotary(x[-1:, -5:].transpose(1, 2).contiguous(), rot, start_idx=T - 5)
    assert torch.equal(y[-1:, :, -5:], want)
    n, _ = tb.qk_norm_rotary(x.transpose(1, 2), x.transpose(1, 2), rot=rot)
    want, _ = tb.qk_norm_rotary(x[-1:, -5:].transpose(1, 2), x[-1:, -5:].transpose(1, 2), rot=rot, start_idx=T - 5)
    assert torch.equal(n[-1:, :, -5:], want)
