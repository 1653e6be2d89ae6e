"""CPU-only checks of the gated linear recurrence's entry points: sizes, refusals, and the oracle's own gradients."""

import ctypes as C

import pytest
import torch

from oracle import gated_oracle as O
from ttt_rs_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from ttt_rs_b200.build import build
    build()
    return _lib.load()


def dims(**kw):
    return _lib.TttDims(**{**dict(batch=2, heads=3, seq_len=100, head_dim=64, mini_batch=0, checkpoint_interval=0, epsilon=0.0,
                                  dtype=1), **kw})


FAKE = C.c_void_p(0x1000)


def forward(lib, d, strides=None, saved=None, saved_bytes=0, ws=None, ws_bytes=0, **at):
    names = ("xq", "xk", "xv", "log_decay", "beta", "weight", "output", "weight_out")
    p = {n: at.get(n, FAKE) for n in names}
    s = None if strides is None else C.cast((C.c_int64 * 9)(*strides), C.c_void_p)
    return lib.ttt_linear_gated_forward(C.byref(d), p["xq"], p["xk"], p["xv"], s, p["log_decay"], p["beta"], p["weight"],
                                        p["output"], p["weight_out"], saved, saved_bytes, ws, ws_bytes, None, None)


def test_sizes(lib):
    assert lib.ttt_linear_gated_saved_bytes(C.byref(dims())) == 6 * 2 * 64 * 64 * 4
    assert lib.ttt_linear_gated_saved_bytes(C.byref(dims(head_dim=32, seq_len=64))) == 6 * 32 * 32 * 4
    many = dims(batch=32, heads=12, seq_len=2048)
    assert lib.ttt_linear_gated_forward_workspace_bytes(C.byref(many)) == 0
    # more streams than blocks are resident: a state and a flag per range, and the counter
    assert lib.ttt_linear_gated_backward_workspace_bytes(C.byref(many)) == 296 * (64 * 64 + 1) * 4 + 4
    assert lib.ttt_linear_gated_backward_workspace_bytes(C.byref(dims(batch=16, heads=16, seq_len=2048))) == 0
    few = lib.ttt_linear_gated_forward_workspace_bytes(C.byref(dims(batch=1, heads=1, seq_len=8192)))
    assert few > 0 and few % (64 * 64 * 4 + 4) == 0  # a state and a decay per segment
    for bad in (dict(head_dim=48), dict(batch=0), dict(seq_len=0), dict(dtype=3)):
        assert lib.ttt_linear_gated_saved_bytes(C.byref(dims(**bad))) == 0
        assert lib.ttt_linear_gated_backward_workspace_bytes(C.byref(dims(**bad))) == 0


def test_refusals(lib):
    assert forward(lib, dims(head_dim=48)) == _lib.TTT_ERR_UNSUPPORTED
    assert forward(lib, dims(dtype=2)) == _lib.TTT_ERR_UNSUPPORTED
    assert forward(lib, dims(seq_len=0)) == forward(lib, dims(heads=0)) == _lib.TTT_ERR_SHAPE
    assert forward(lib, dims(seq_len=1 << 30)) == _lib.TTT_ERR_SHAPE
    for n in ("xq", "xk", "xv", "log_decay", "output", "weight_out"):
        assert forward(lib, dims(), **{n: None}) == _lib.TTT_ERR_NULL and n in _lib.last_error()
    for n in ("xq", "output", "weight"):
        assert forward(lib, dims(), **{n: C.c_void_p(0x1008)}) == _lib.TTT_ERR_ALIGN and n in _lib.last_error()
    assert forward(lib, dims(), log_decay=C.c_void_p(0x1002)) == _lib.TTT_ERR_ALIGN
    assert forward(lib, dims(), saved=FAKE, saved_bytes=100) == _lib.TTT_ERR_WORKSPACE
    few = dims(batch=1, heads=1, seq_len=8192)
    assert forward(lib, few) == _lib.TTT_ERR_WORKSPACE
    assert forward(lib, few, ws=FAKE, ws_bytes=16) == _lib.TTT_ERR_WORKSPACE
    need = lib.ttt_linear_gated_forward_workspace_bytes(C.byref(few))
    assert forward(lib, few, ws=C.c_void_p(0x1004), ws_bytes=need) == _lib.TTT_ERR_ALIGN
    dense = [3 * 6400, 6400, 64]
    for bad in ([3 * 6400, 6400, 68], [3 * 6400, 0, 64], [3 * 6400, -6400, 64]):
        assert forward(lib, dims(), strides=dense + bad + dense) == _lib.TTT_ERR_ALIGN and "xk" in _lib.last_error()


def test_backward_and_step_refuse(lib):
    def backward(d=None, **at):
        names = ("xq", "xk", "xv", "grad_output", "strides", "log_decay", "beta", "saved", "bytes", "grad_weight_out", "grad_xq",
                 "grad_xk", "grad_xv", "grad_log_decay", "grad_beta", "grad_weight")
        p = {**{n: FAKE for n in names}, "strides": None, "bytes": 1 << 30, "grad_weight_out": None, **at}
        return lib.ttt_linear_gated_backward(C.byref(d or dims()), *[p[n] for n in names], None, 0, None, None)

    assert backward(bytes=16) == _lib.TTT_ERR_WORKSPACE
    assert backward(saved=None) == backward(grad_xk=None) == backward(grad_log_decay=None) == _lib.TTT_ERR_NULL
    assert backward(beta=None) == backward(grad_beta=None) == _lib.TTT_ERR_NULL
    assert backward(grad_weight_out=C.c_void_p(0x1004)) == _lib.TTT_ERR_ALIGN
    assert backward(dims(batch=1, heads=1, seq_len=8192)) == _lib.TTT_ERR_WORKSPACE
    step = lambda d, **at: lib.ttt_linear_gated_step(C.byref(d), FAKE, FAKE, FAKE, None, at.get("g", FAKE), None, None,  # noqa: E731
                                                     FAKE, at.get("w", FAKE), None)
    assert step(dims(seq_len=17)) == step(dims(seq_len=0)) == _lib.TTT_ERR_SHAPE
    assert step(dims(seq_len=1), g=None) == step(dims(seq_len=1), w=None) == _lib.TTT_ERR_NULL
    assert step(dims(seq_len=1), w=C.c_void_p(0x1004)) == _lib.TTT_ERR_ALIGN


def test_host_refuses_cpu_tensors():
    import ttt_rs_b200 as tb
    x = torch.zeros(1, 1, 4, 64)
    with pytest.raises(tb.TttError):
        tb.fused_gated_linear(x, x, x, torch.zeros(1, 1, 4))


def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    ins = [torch.randn(1, 2, 6, 4, generator=g, dtype=torch.float64) for _ in range(3)]
    ins += [-torch.rand(1, 2, 6, generator=g, dtype=torch.float64), torch.rand(1, 2, 6, generator=g, dtype=torch.float64),
            torch.randn(1, 2, 4, 4, generator=g, dtype=torch.float64)]
    assert torch.autograd.gradcheck(O.gated_forward, [t.requires_grad_() for t in ins])
