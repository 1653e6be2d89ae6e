"""CPU-only checks of the rotary entry points: configurations, the table of turns, and refusals of the C ABI."""

import ctypes as C
import math

import pytest
import torch

from oracle import rotary_oracle as O
from ttt_rs_b200 import _lib
from ttt_rs_b200.rope import Rotary, RotaryConfig


@pytest.fixture(scope="module")
def lib():
    from ttt_rs_b200.build import build
    build()
    return _lib.load()


@pytest.mark.parametrize("kw", [dict(), dict(rotary_dim=24), dict(theta=500000.0), dict(scaling="linear", factor=4.0),
                                dict(scaling="ntk", factor=4.0), dict(scaling="by_parts", factor=16.0, original_length=8192)])
@pytest.mark.parametrize("pos", [0, 1, 12345, -7, (1 << 20) + 1, 1 << 33])
def test_table_gives_the_angle_of_any_position(kw, pos):
    """position * turns modulo 2^64, as the kernel multiplies.  Both frequencies are doubles: the table's is a power (off by a few
    2^-53 of itself), the oracle's exp(y) with y = 2p / r log(theta') up to 14, whose own roundings (of the logarithm, the quotient
    and the product: 3 y 2^-53) shift the result by up to 42 * 2^-53 of itself; with the scaling's factors below 2^-46 in all."""
    cfg = RotaryConfig(head_dim=64, **kw)
    turns = Rotary(cfg, device="cpu").turns.tolist()
    want, size = O.angles(cfg, torch.tensor([pos]))
    assert size == pytest.approx(cfg.size)
    for t, f, a in zip(turns, cfg.frequencies(), want[0].tolist()):
        got = ((pos * t) % 2 ** 64) / 2 ** 64
        off = (got - a / (2 * math.pi) + 0.5) % 1.0 - 0.5
        assert abs(off) <= abs(pos * f) * 2 ** -46 + 2 ** -60


def test_scalings_meet_their_definitions():
    base = RotaryConfig(head_dim=64).frequencies()
    lin = RotaryConfig(head_dim=64, scaling="linear", factor=8.0).frequencies()
    ntk = RotaryConfig(head_dim=64, scaling="ntk", factor=8.0).frequencies()
    parts = RotaryConfig(head_dim=64, scaling="by_parts", factor=8.0, original_length=4096).frequencies()
    assert all(x == pytest.approx(y / 8) for x, y in zip(lin, base))
    assert ntk[0] == base[0] and ntk[-1] == pytest.approx(base[-1] / 8)
    assert parts[0] == base[0] and parts[-1] == pytest.approx(base[-1] / 8)
    assert all(y / 8 * (1 - 1e-12) <= x <= y for x, y in zip(parts, base))


@pytest.mark.parametrize("kw", [dict(head_dim=63), dict(head_dim=258), dict(rotary_dim=66), dict(rotary_dim=3), dict(rotary_dim=0),
                                dict(theta=0.5), dict(theta=math.inf), dict(layout="other"), dict(scaling="other"),
                                dict(scaling="linear", factor=0.5), dict(scaling="by_parts", factor=2.0), dict(wrap=-1),
                                dict(scaling="ntk", factor=2.0, rotary_dim=2)])
def test_bad_configurations(kw):
    with pytest.raises(ValueError):
        RotaryConfig(**{"head_dim": 64, **kw})


FAKE = C.c_void_p(0x1000)


def dims(**kw):
    return _lib.TttDims(**{**dict(batch=2, heads=3, seq_len=10, head_dim=64, mini_batch=0, checkpoint_interval=0, epsilon=1e-6, dtype=1), **kw})


def rotation(**kw):
    return _lib.TttRotation(**{**dict(turns=0x1000, positions=None, positions_stride=0, start_idx=0, rotary_dim=64, half=0, wrap=0, size=1.0), **kw})


def test_rotary_refuses(lib):
    def call(d=None, rot=None, x=FAKE, y=FAKE, ys=None, xs=None):
        arr = lambda s: None if s is None else C.cast((C.c_int64 * 3)(*s), C.c_void_p)  # noqa: E731
        return lib.ttt_layer_rotary(C.byref(d or dims()), x, arr(xs), C.byref(rot or rotation()), 0, y, arr(ys), None)

    for bad in (dict(head_dim=63), dict(head_dim=258), dict(dtype=2)):
        assert call(dims(**bad)) == _lib.TTT_ERR_UNSUPPORTED
    assert call(dims(seq_len=0)) == call(dims(batch=-1)) == _lib.TTT_ERR_SHAPE
    for bad in (dict(rotary_dim=66), dict(rotary_dim=5), dict(wrap=-1), dict(size=0.0), dict(positions=0x1000, positions_stride=4)):
        assert call(rot=rotation(**bad)) == _lib.TTT_ERR_SHAPE, bad
    assert call(rot=rotation(half=2)) == _lib.TTT_ERR_UNSUPPORTED
    assert call(rot=rotation(turns=None)) == call(x=None) == call(y=None) == _lib.TTT_ERR_NULL
    assert lib.ttt_layer_rotary(C.byref(dims()), FAKE, None, None, 0, FAKE, None, None) == _lib.TTT_ERR_NULL
    assert call(x=C.c_void_p(0x1001)) == call(rot=rotation(turns=0x1004)) == _lib.TTT_ERR_ALIGN
    assert call(ys=[1920, 640, 0]) == call(xs=[-1, 640, 64]) == _lib.TTT_ERR_SHAPE


def test_qk_norm_refuses(lib):
    def call(d=None, k_heads=3, rot=None, **at):
        p = {**{n: FAKE for n in ("q", "k", "wq", "wk", "yq", "yk")}, **at}
        return lib.ttt_layer_qk_norm_rotary(C.byref(d or dims()), k_heads, p["q"], p["k"], None, p["wq"], p["wk"],
                                            C.byref(rot or rotation()), p["yq"], p["yk"], None, None)

    assert call(k_heads=0) == call(k_heads=-1) == call(dims(epsilon=-1.0)) == call(dims(epsilon=float("nan"))) == _lib.TTT_ERR_SHAPE
    assert call(dims(heads=65535), 1) == _lib.TTT_ERR_UNSUPPORTED
    for n in ("q", "k", "yq", "yk"):
        assert call(**{n: None}) == _lib.TTT_ERR_NULL
    assert call(wq=C.c_void_p(0x1001)) == _lib.TTT_ERR_ALIGN
    assert lib.ttt_layer_qk_norm_rotary_backward_workspace_bytes(C.byref(dims()), 0) == 0
    need = lib.ttt_layer_qk_norm_rotary_backward_workspace_bytes(C.byref(dims()), 3)
    assert need > 0 and need % (2 * 64 * 4) == 0

    def backward(ws=FAKE, ws_bytes=need, **at):
        names = ("q", "k", "gq", "gk", "strides", "wq", "wk", "rot", "dq", "dk", "dstrides", "dwq", "dwk")
        p = {**{n: FAKE for n in names}, "strides": None, "dstrides": None, "rot": C.byref(rotation()), **at}
        return lib.ttt_layer_qk_norm_rotary_backward(C.byref(dims()), 3, *[p[n] for n in names], ws, ws_bytes, None)

    assert backward(ws_bytes=need - 4) == backward(ws=None) == _lib.TTT_ERR_WORKSPACE
    assert backward(gq=None) == backward(dk=None) == _lib.TTT_ERR_NULL
    assert backward(dwq=C.c_void_p(0x1001)) == _lib.TTT_ERR_ALIGN


@pytest.mark.parametrize("strides", [(192, 64, 64), (640, 640, 64), (1920, 640, 1), (1919, 640, 64), (128, 256, 800), (1 << 61, 640, 64)])
def test_rows_of_a_result_must_not_overlap(lib, strides):
    rot = rotation()
    ys = (C.c_int64 * 3)(*strides)
    assert lib.ttt_layer_rotary(C.byref(dims(batch=3)), FAKE, None, C.byref(rot), 0, FAKE, ys, None) == _lib.TTT_ERR_SHAPE
