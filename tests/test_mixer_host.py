"""CPU-only checks of the selective layer's entry points: sizes, refusals, the oracles' own gradients."""

import ctypes as C

import pytest
import torch

import ttt_rs_b200 as tb
from oracle import mixer_oracle as O
from ttt_rs_b200 import _lib

FAKE = C.c_void_p(0x100000)


@pytest.fixture(scope="module")
def lib():
    from ttt_rs_b200.build import build
    build()
    return _lib.load()


def at(address):
    return C.c_void_p(address)


def int64s(*v):
    return C.cast((C.c_int64 * len(v))(*v), C.c_void_p)


def test_convolution_refuses(lib):
    def conv(B=2, T=9, Ch=16, K=4, dtype=1, act=1, strides=None, **p):
        d = dict(x=0x100000, weight=0x200000, bias=None, state=0x300000, starts=None, y=0x400000, state_out=0x500000)
        d.update(p)
        return lib.ttt_layer_causal_conv(B, T, Ch, K, dtype, act, d["x"], strides, *[d[n] for n in ("weight", "bias", "state", "starts", "y",
                                                                                                    "state_out")], None)
    assert conv(B=0) == conv(T=0) == conv(Ch=0) == conv(B=1 << 20, T=1 << 20) == _lib.TTT_ERR_SHAPE
    assert conv(K=1) == conv(K=5) == conv(dtype=2) == conv(act=2) == conv(Ch=1 << 21) == _lib.TTT_ERR_UNSUPPORTED
    for n in ("x", "weight", "y", "state_out"):
        assert conv(**{n: None}) == _lib.TTT_ERR_NULL and n in _lib.last_error()
    for n in ("x", "weight", "y", "state_out", "state", "bias"):
        assert conv(**{n: 0x600001}) == _lib.TTT_ERR_ALIGN and n in _lib.last_error()
    assert conv(strides=int64s(144, -16)) == conv(strides=int64s(1 << 60, 16)) == _lib.TTT_ERR_SHAPE
    # the new state over part of the given one, or over another tensor
    for n in (dict(state_out=0x300002), dict(state_out=0x100000), dict(state_out=0x400010), dict(state_out=0x200000), dict(y=0x100010),
              dict(y=0x300000)):
        assert conv(**n) == _lib.TTT_ERR_SHAPE and "lies over" in _lib.last_error()


def test_convolution_backward_refuses(lib):
    need = lib.ttt_layer_causal_conv_backward_workspace_bytes(2, 9, 16, 4, 1)
    assert need > 0 and lib.ttt_layer_causal_conv_backward_workspace_bytes(2, 9, 16, 5, 1) == 0

    def back(ws=FAKE, bytes_=need, **p):
        names = ("weight", "bias", "state", "starts", "grad_state_out", "grad_x", "grad_weight", "grad_bias", "grad_state")
        d = {**{n: FAKE for n in names}, "x": FAKE, "grad_y": FAKE, **p}
        return lib.ttt_layer_causal_conv_backward(2, 9, 16, 4, 1, 1, d["x"], d["grad_y"], None, *[d[n] for n in names], ws, bytes_, None)
    assert back(bytes_=need - 1) == back(ws=None) == _lib.TTT_ERR_WORKSPACE
    assert back(ws=at(0x100004)) == back(grad_x=at(0x100001)) == _lib.TTT_ERR_ALIGN
    assert back(x=None) == back(grad_y=None) == back(grad_x=None) == back(weight=None) == _lib.TTT_ERR_NULL


def test_norm_refuses(lib):
    def norm(B=2, T=9, Ch=32, G=4, over=0, dtype=1, act=1, eps=1e-5, ws=FAKE, bytes_=1 << 20, strides=None, **p):
        d = dict(x=FAKE, gate=FAKE, weight=FAKE, bias=FAKE, y=FAKE, stats=FAKE)
        d.update(p)
        return lib.ttt_layer_group_norm(B, T, Ch, G, over, dtype, act, eps, d["x"], d["gate"], strides, d["weight"], d["bias"], d["y"],
                                        d["stats"], ws, bytes_, None)
    assert norm(G=5) == norm(G=0) == norm(T=0) == norm(eps=-1.0) == norm(eps=float("nan")) == _lib.TTT_ERR_SHAPE
    assert norm(over=2) == norm(act=3) == norm(dtype=5) == norm(Ch=8192, G=1) == _lib.TTT_ERR_UNSUPPORTED
    assert norm(over=1, bytes_=4) == norm(over=1, ws=None) == _lib.TTT_ERR_WORKSPACE
    assert norm(x=None) == norm(y=None) == _lib.TTT_ERR_NULL
    assert norm(gate=at(0x100001)) == norm(weight=at(0x100001)) == norm(stats=at(0x100002)) == _lib.TTT_ERR_ALIGN
    assert norm(strides=int64s(288, 32, -1, 32)) == _lib.TTT_ERR_SHAPE

    def back(over=0, ws=FAKE, bytes_=1 << 24, **p):
        d = dict(x=FAKE, gate=FAKE, grad_y=FAKE, weight=FAKE, bias=FAKE, stats=FAKE, grad_x=FAKE, grad_gate=FAKE, grad_weight=FAKE, grad_bias=FAKE)
        d.update(p)
        return lib.ttt_layer_group_norm_backward(2, 9, 32, 4, over, 1, 1, 1e-5, d["x"], d["gate"], d["grad_y"], None, d["weight"], d["bias"],
                                                 d["stats"], d["grad_x"], d["grad_gate"], d["grad_weight"], d["grad_bias"], ws, bytes_, None)
    assert back(grad_gate=None) == back(grad_x=None) == back(grad_y=None) == back(over=1, stats=None) == _lib.TTT_ERR_NULL
    assert back(bytes_=8) == back(ws=None) == back(over=1, bytes_=8, grad_weight=None, grad_bias=None) == _lib.TTT_ERR_WORKSPACE


def test_scan_refuses(lib):
    def scan(B=2, T=40, Ch=32, G=2, N=16, dtype=1, strides=None, ws=None, bytes_=0, saved=None, saved_bytes=0, **p):
        names = ("x", "dt", "a", "b", "c", "d", "z", "dt_bias", "state", "starts")
        d = {n: 0x100000 * (i + 1) for i, n in enumerate(names)} | {"starts": None, "y": 0x2000000, "state_out": 0x3000000} | p
        return lib.ttt_linear_selective_forward(B, T, Ch, G, N, dtype, 1, *[d[n] for n in names], strides, d["y"], d["state_out"], saved, saved_bytes,
                                                ws, bytes_, None)
    assert scan(G=5) == scan(G=0) == scan(T=0) == scan(B=0) == scan(B=1 << 11, Ch=1 << 20, G=1) == _lib.TTT_ERR_SHAPE
    assert scan(N=0) == scan(N=65) == scan(dtype=3) == _lib.TTT_ERR_UNSUPPORTED
    for n in ("x", "dt", "a", "b", "c", "y", "state_out"):
        assert scan(**{n: None}) == _lib.TTT_ERR_NULL and n in _lib.last_error()
    for n in ("x", "dt", "z", "b", "c", "y", "d", "dt_bias"):
        assert scan(**{n: 0x4000001}) == _lib.TTT_ERR_ALIGN and n in _lib.last_error()
    for n in ("a", "state", "state_out"):
        assert scan(**{n: 0x4000008}) == _lib.TTT_ERR_ALIGN and n in _lib.last_error()
    dense = [40 * 32, 32] * 3 + [40 * 32, 32, 16] * 2
    for i, bad in ((0, -1), (3, 1 << 60), (8, -16)):
        s = list(dense)
        s[i] = bad
        assert scan(strides=int64s(*s)) == _lib.TTT_ERR_SHAPE
    assert scan(saved=FAKE, saved_bytes=8) == _lib.TTT_ERR_WORKSPACE
    need = lib.ttt_linear_selective_forward_workspace_bytes(2, 40, 32, 2, 16, 1)
    if need:
        assert scan(ws=FAKE, bytes_=need - 1) == _lib.TTT_ERR_WORKSPACE and scan(ws=at(0x100008), bytes_=need) == _lib.TTT_ERR_ALIGN
    # results over other tensors of the call
    for n in (dict(state_out=0x900010), dict(state_out=0x100000), dict(state_out=0x300000), dict(state_out=0x2000000), dict(y=0x100000),
              dict(y=0x900000), dict(y=0x400000)):
        assert scan(**n) == _lib.TTT_ERR_SHAPE and "lies over" in _lib.last_error(), n


def test_scan_backward_refuses(lib):
    shape = (2, 40, 32, 2, 16, 1)
    saved, need = lib.ttt_linear_selective_saved_bytes(*shape), lib.ttt_linear_selective_backward_workspace_bytes(*shape)
    assert saved == 2 * 3 * 32 * 16 * 4 and need > 0
    assert lib.ttt_linear_selective_saved_bytes(2, 40, 32, 5, 16, 1) == lib.ttt_linear_selective_backward_workspace_bytes(2, 40, 32, 2, 65, 1) == 0

    def back(ws=FAKE, bytes_=need, saved_bytes=saved, **p):
        first = ("x", "dt", "a", "b", "c", "d", "z", "dt_bias", "starts", "grad_y")
        last = ("grad_state_out", "grad_x", "grad_dt", "grad_a", "grad_b", "grad_c", "grad_d", "grad_z", "grad_dt_bias", "grad_state")
        d = {**{n: FAKE for n in first + last}, "saved": FAKE, **p}
        return lib.ttt_linear_selective_backward(*shape, 1, *[d[n] for n in first], None, d["saved"], saved_bytes, *[d[n] for n in last], ws, bytes_,
                                                 None)
    assert back(bytes_=need - 1) == back(ws=None) == back(saved_bytes=16) == _lib.TTT_ERR_WORKSPACE
    for n in ("grad_y", "grad_x", "grad_dt", "grad_z", "grad_a", "grad_b", "grad_c", "saved"):
        assert back(**{n: None}) == _lib.TTT_ERR_NULL and n in _lib.last_error()
    for n in ("grad_a", "grad_state", "grad_state_out"):
        assert back(**{n: at(0x100008)}) == _lib.TTT_ERR_ALIGN and n in _lib.last_error()
    assert back(ws=at(0x100004)) == back(grad_b=at(0x100001)) == back(grad_d=at(0x100002)) == _lib.TTT_ERR_ALIGN


def test_host_refuses_cpu_tensors():
    x = torch.zeros(1, 4, 16)
    b = torch.zeros(1, 4, 8)
    for f in (lambda: tb.causal_conv(x, torch.zeros(16, 4)), lambda: tb.group_norm(x, 4), lambda: tb.selective_scan(x, x, torch.zeros(16, 8), b, b)):
        with pytest.raises(tb.TttError):
            f()


def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()  # noqa: E731
    marks = torch.tensor([[False, True, False, False, False], [False, False, False, True, False]])
    assert torch.autograd.gradcheck(lambda *t: O.causal_conv(*t, activation="silu", starts=marks), [r(2, 5, 3), r(3, 4), r(3), r(2, 3, 3)])
    assert torch.autograd.gradcheck(lambda *t: O.group_norm(t[0], 2, t[1], t[2], gate=t[3], activation="silu"), [r(2, 3, 6), r(6), r(6), r(2, 3, 6)])
    assert torch.autograd.gradcheck(lambda *t: O.group_norm(t[0], 2, t[1], t[2], activation="gelu", over="sequence"), [r(2, 3, 6), r(6), r(6)])
    assert torch.autograd.gradcheck(
        lambda x, dt, A, B, C, D, z, bias, h: O.selective_scan(x, dt, A, B, C, D, z, bias, h, starts=marks),
        [r(2, 5, 4), r(2, 5, 4), r(4, 3), r(2, 5, 2, 3), r(2, 5, 2, 3), r(4), r(2, 5, 4), r(4), r(2, 4, 3)])
