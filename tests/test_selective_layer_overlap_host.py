"""CPU-only: results of the selective layer's C entry points that lie over other tensors of the call are refused before anything is launched."""

import ctypes as C

import pytest

from ttt_rs_b200 import _lib

MB = 1 << 20


@pytest.fixture(scope="module")
def lib():
    from ttt_rs_b200.build import build
    build()
    return _lib.load()


def places(names):
    """A megabyte of its own for each, 16-byte aligned."""
    return {n: (i + 1) * MB for i, n in enumerate(names)}


def refused(call, d, **over):
    p = dict(d)
    p.update(over)
    rc = call(p)
    return rc == _lib.TTT_ERR_SHAPE and "lies over" in _lib.last_error()


def each_pair(call, d, results, inputs, sizes, may=()):
    """Every result over the first and the last bytes of every other tensor; `may`: pairs that may be the same."""
    for r in results:
        for o in (*inputs, *results):
            if o == r:
                continue
            if (r, o) not in may and (o, r) not in may:
                assert refused(call, d, **{r: d[o]}), (r, o)
            assert refused(call, d, **{r: d[o] + (sizes[o] - 1) // 16 * 16}), (r, o, "end")  # (sizes above 16)
            assert refused(call, d, **{r: d[o] - (sizes[r] - 1) // 16 * 16}), (r, o, "start")


def test_convolution(lib):
    B, T, Ch, K = 2, 9, 16, 4
    n, held = B * T * Ch * 2, B * (K - 1) * Ch * 2
    sizes = dict(x=n, weight=Ch * K * 2, bias=Ch * 2, state=held, starts=B * T, y=n, state_out=held)
    d = places(sizes)
    call = lambda p: lib.ttt_layer_causal_conv(B, T, Ch, K, 1, 1, p["x"], None, *[p[k] for k in ("weight", "bias", "state", "starts", "y", "state_out")], None)  # noqa: E731
    each_pair(call, d, ("y", "state_out"), ("x", "weight", "bias", "state", "starts"), sizes, may=[("state_out", "state")])


def test_convolution_backward(lib):
    B, T, Ch, K = 2, 9, 16, 4
    need = lib.ttt_layer_causal_conv_backward_workspace_bytes(B, T, Ch, K, 1)
    n, held, w = B * T * Ch * 2, B * (K - 1) * Ch * 2, Ch * K * 2
    ins = dict(x=n, grad_y=n, weight=w, bias=Ch * 2, state=held, starts=B * T, grad_state_out=held)
    outs = dict(grad_x=n, grad_weight=w, grad_bias=Ch * 2, grad_state=held, workspace=need)
    d = places({**ins, **outs})

    def call(p):
        return lib.ttt_layer_causal_conv_backward(B, T, Ch, K, 1, 1, p["x"], p["grad_y"], None, *[p[k] for k in (
            "weight", "bias", "state", "starts", "grad_state_out", "grad_x", "grad_weight", "grad_bias", "grad_state")], p["workspace"], need, None)
    each_pair(call, d, outs, ins, {**ins, **outs}, may=[("grad_state", "state"), ("grad_weight", "weight"), ("grad_bias", "bias")])


@pytest.mark.parametrize("over", [0, 1])
def test_norm(lib, over):
    B, T, Ch, G = 2, 9, 32, 4
    need = lib.ttt_layer_group_norm_workspace_bytes(B, T, Ch, G, over, 1)
    n, stats = B * T * Ch * 2, B * G * 8
    sizes = dict(x=n, gate=n, weight=Ch * 2, bias=Ch * 2, y=n, stats=stats, workspace=need)
    d = places(sizes)
    strides = None

    def call(p):
        return lib.ttt_layer_group_norm(B, T, Ch, G, over, 1, 1, 1e-5, p["x"], p["gate"], strides, p["weight"], p["bias"], p["y"], p["stats"],
                                        p["workspace"], need, None)
    results = ("y", "stats", "workspace") if over else ("y",)
    each_pair(call, d, results, ("x", "gate", "weight", "bias"), sizes, may=[("y", "x"), ("y", "gate")])
    # the same bytes in another order: batch and token exchanged
    strides = C.cast((C.c_int64 * 4)(Ch, B * Ch, T * Ch, Ch), C.c_void_p)
    assert refused(call, d, y=d["x"])


@pytest.mark.parametrize("over", [0, 1])
def test_norm_backward(lib, over):
    B, T, Ch, G = 2, 9, 32, 4
    need = lib.ttt_layer_group_norm_backward_workspace_bytes(B, T, Ch, G, over, 1)
    n, stats = B * T * Ch * 2, B * G * 8
    ins = dict(x=n, gate=n, grad_y=n, weight=Ch * 2, bias=Ch * 2, **(dict(stats=stats) if over else {}))
    outs = dict(grad_x=n, grad_gate=n, grad_weight=Ch * 2, grad_bias=Ch * 2, workspace=need)
    d = places({**ins, **outs})

    def call(p):
        return lib.ttt_layer_group_norm_backward(B, T, Ch, G, over, 1, 1, 1e-5, p["x"], p["gate"], p["grad_y"], None, p["weight"], p["bias"],
                                                 p.get("stats"), p["grad_x"], p["grad_gate"], p["grad_weight"], p["grad_bias"], p["workspace"], need, None)
    may = [(r, i) for r in ("grad_x", "grad_gate") for i in ("x", "gate", "grad_y")] + [("grad_weight", "weight"), ("grad_bias", "bias")]
    each_pair(call, d, outs, ins, {**ins, **outs}, may=may)


@pytest.mark.parametrize("T", [9, 700])
def test_scan(lib, T):
    shape = B, _, Ch, G, N, dt = 2, T, 32, 2, 16, 1
    need = lib.ttt_linear_selective_forward_workspace_bytes(*shape) if T > 16 else 0
    assert (need > 0) == (T > 16)
    n, bc, state = B * T * Ch * 2, B * T * G * N * 2, B * Ch * N * 4
    ins = dict(x=n, dt=n, a=Ch * N * 4, b=bc, c=bc, d=Ch * 4, z=n, dt_bias=Ch * 4, state=state, starts=B * T)
    saved = lib.ttt_linear_selective_saved_bytes(*shape) if T > 16 else 0
    outs = dict(y=n, state_out=state, **(dict(saved=saved, workspace=need) if T > 16 else {}))
    d = places({**ins, **outs})

    def call(p):
        return lib.ttt_linear_selective_forward(*shape, 1, *[p[k] for k in ins], None, p["y"], p["state_out"], p.get("saved"), saved, p.get("workspace"),
                                                need, None)
    each_pair(call, d, outs, ins, {**ins, **outs}, may=[("state_out", "state")])


def test_scan_backward(lib):
    shape = B, T, Ch, G, N, dt = 2, 700, 32, 2, 16, 1
    need, saved = lib.ttt_linear_selective_backward_workspace_bytes(*shape), lib.ttt_linear_selective_saved_bytes(*shape)
    n, bc, state, wide = B * T * Ch * 2, B * T * G * N * 2, B * Ch * N * 4, Ch * 4
    ins = dict(x=n, dt=n, a=wide * N, b=bc, c=bc, d=wide, z=n, dt_bias=wide, starts=B * T, grad_y=n, saved=saved, grad_state_out=state)
    outs = dict(grad_x=n, grad_dt=n, grad_a=wide * N, grad_b=bc, grad_c=bc, grad_d=wide, grad_z=n, grad_dt_bias=wide, grad_state=state, workspace=need)
    d = places({**ins, **outs})

    def call(p):
        first = [p[k] for k in ("x", "dt", "a", "b", "c", "d", "z", "dt_bias", "starts", "grad_y")]
        last = [p[k] for k in ("grad_state_out", "grad_x", "grad_dt", "grad_a", "grad_b", "grad_c", "grad_d", "grad_z", "grad_dt_bias", "grad_state")]
        return lib.ttt_linear_selective_backward(*shape, 1, *first, None, p["saved"], saved, *last, p["workspace"], need, None)
    may = [(r, i) for r in ("grad_x", "grad_dt", "grad_z") for i in ("x", "dt", "z", "grad_y")] + [(r, i) for r in ("grad_b", "grad_c") for i in ("b", "c")]
    may += [("grad_a", "a"), ("grad_d", "d"), ("grad_dt_bias", "dt_bias")]
    each_pair(call, d, outs, ins, {**ins, **outs}, may=may)
