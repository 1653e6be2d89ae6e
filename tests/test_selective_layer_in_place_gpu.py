"""C entry points of the selective layer's operators with results in the place of tensors that may be them: the same as apart."""

import ctypes as C

import pytest
import torch

from ttt_rs_b200 import _lib

pytestmark = pytest.mark.gpu


def run(f, order, tensors, place):
    """f's results by name; place: result -> input in whose place it goes.  f takes addresses by name."""
    t = {k: v.clone() for k, v in tensors.items()}
    for r, i in place.items():
        t[r] = t[i]
    torch.cuda.synchronize()
    rc = f({k: C.c_void_p(v.data_ptr()) for k, v in t.items()}, C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == _lib.TTT_OK, _lib.last_error()
    torch.cuda.synchronize()
    return {k: t[k] for k in order}


def check(f, results, tensors, places):
    want = run(f, results, tensors, {})
    for place in places:
        got = run(f, results, tensors, place)
        for k in results:
            assert torch.equal(got[k], want[k]), (place, k)


def rand(dtype, *s):
    return torch.randn(*s, device="cuda").to(dtype)


def space(n, dtype=torch.uint8):
    return torch.zeros(max(int(n), 16), device="cuda", dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("over,c", [(0, 16), (0, 520), (0, 7), (1, 16), (1, 2050)])
def test_norm(over, c, dtype):
    lib, kind = _lib.load(), int(dtype == torch.bfloat16)
    B, T, G = 3, 500, 4 if c < 100 else 1
    shape = (B, T, G * c, G, over, kind)
    need, back = lib.ttt_layer_group_norm_workspace_bytes(*shape), lib.ttt_layer_group_norm_backward_workspace_bytes(*shape)
    t = dict(x=rand(dtype, B, T, G * c), gate=rand(dtype, B, T, G * c), weight=rand(dtype, G * c), bias=rand(dtype, G * c), y=rand(dtype, B, T, G * c),
             stats=space(2 * B * G, torch.float32), ws=space(need))
    f = lambda p, st: lib.ttt_layer_group_norm(*shape, 1, 1e-3, p["x"], p["gate"], None, p["weight"], p["bias"], p["y"], p["stats"], p["ws"], need, st)  # noqa: E731
    check(f, ["y"], t, [dict(y="x"), dict(y="gate")])
    t["stats"] = run(f, ["stats"], t, {})["stats"]
    t |= dict(grad_y=rand(dtype, B, T, G * c), grad_x=rand(dtype, B, T, G * c), grad_gate=rand(dtype, B, T, G * c), grad_weight=rand(dtype, G * c),
              grad_bias=rand(dtype, G * c), ws=space(back))
    check(lambda p, st: lib.ttt_layer_group_norm_backward(*shape, 1, 1e-3, p["x"], p["gate"], p["grad_y"], None, p["weight"], p["bias"], p["stats"], p["grad_x"],
                                                          p["grad_gate"], p["grad_weight"], p["grad_bias"], p["ws"], back, st),
          ["grad_x", "grad_gate", "grad_weight", "grad_bias"], t,
          [dict(grad_x="x", grad_gate="gate"), dict(grad_x="grad_y", grad_weight="weight", grad_bias="bias"), dict(grad_x="gate", grad_gate="grad_y"),
           dict(grad_gate="x")])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,Ch", [(1, 64), (2, 7), (300, 64), (301, 1030)])
def test_convolution_backward(T, Ch, dtype):
    lib, kind = _lib.load(), int(dtype == torch.bfloat16)
    B, K = 3, 4
    need = lib.ttt_layer_causal_conv_backward_workspace_bytes(B, T, Ch, K, kind)
    held = lambda: rand(dtype, B, K - 1, Ch)  # noqa: E731
    t = dict(x=rand(dtype, B, T, Ch), grad_y=rand(dtype, B, T, Ch), weight=rand(dtype, Ch, K), bias=rand(dtype, Ch), state=held(), grad_state_out=held(),
             grad_x=rand(dtype, B, T, Ch), grad_weight=rand(dtype, Ch, K), grad_bias=rand(dtype, Ch), grad_state=held(), ws=space(need))
    results = ["grad_x", "grad_weight", "grad_bias", "grad_state"]
    check(lambda p, st: lib.ttt_layer_causal_conv_backward(B, T, Ch, K, kind, 1, p["x"], p["grad_y"], None, p["weight"], p["bias"], p["state"], None,
                                                           p["grad_state_out"], *[p[k] for k in results], p["ws"], need, st),
          results, t, [dict(grad_weight="weight", grad_bias="bias", grad_state="state")])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,Ch,N", [(9, 64, 16), (700, 96, 16), (300, 40, 4)])
def test_scan_backward(T, Ch, N, dtype):
    lib, kind = _lib.load(), int(dtype == torch.bfloat16)
    B, G = 3, 2
    shape = (B, T, Ch, G, N, kind)
    sizes = [getattr(lib, f"ttt_linear_selective_{n}_bytes")(*shape) for n in ("saved", "forward_workspace", "backward_workspace")]
    rows, bc, f32 = lambda: rand(dtype, B, T, Ch), lambda: rand(dtype, B, T, G, N), torch.float32  # noqa: E731
    t = dict(x=rows(), dt=rows(), a=-torch.rand(Ch, N, device="cuda"), b=bc(), c=bc(), d=rand(f32, Ch), z=rows(), dt_bias=rand(f32, Ch), state=rand(f32, B, Ch, N),
             starts=(torch.rand(B, T, device="cuda") < 0.02).byte(), y=rows(), state_out=rand(f32, B, Ch, N), saved=space(sizes[0]), ws=space(sizes[1]))
    ins = ("x", "dt", "a", "b", "c", "d", "z", "dt_bias")
    t["saved"] = run(lambda p, st: lib.ttt_linear_selective_forward(*shape, 1, *[p[k] for k in ins], p["state"], p["starts"], None, p["y"], p["state_out"],
                                                                    p["saved"], sizes[0], p["ws"], sizes[1], st), ["saved"], t, {})["saved"]
    t |= dict(grad_y=rows(), grad_state_out=rand(f32, B, Ch, N), ws=space(sizes[2]), **{"grad_" + k: torch.empty_like(t[k]) for k in (*ins, "state")})
    results = ["grad_" + k for k in (*ins, "state")]
    check(lambda p, st: lib.ttt_linear_selective_backward(*shape, 1, *[p[k] for k in ins], p["starts"], p["grad_y"], None, p["saved"], sizes[0],
                                                          p["grad_state_out"], *[p[k] for k in results], p["ws"], sizes[2], st),
          results, t, [{"grad_" + k: k for k in ins}, dict(grad_x="grad_y", grad_dt="x", grad_b="c", grad_c="b"), dict(grad_z="dt")])
