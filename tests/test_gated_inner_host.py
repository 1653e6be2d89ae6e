"""CPU-only checks of the gated recurrence's parameter holder."""

import pytest
import torch

import ttt_rs_b200 as tb


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_and_gates_are_float32_whatever_the_model_was_cast_to(dtype):
    inner = tb.FusedGatedLinear(tb.GatedLinear(3, 32)).to(dtype)
    state = inner.init_state(2)
    assert state.weight.dtype == torch.float32 and state.weight.shape == (2, 3, 32, 32) and state.weight.is_contiguous()
    assert torch.equal(state.weight[1], inner.inner.weight_init.float())
    assert state.weight.data_ptr() != inner.inner.weight_init.data_ptr()
    state.weight.sum().backward()
    assert inner.inner.weight_init.grad.dtype == dtype and (inner.inner.weight_init.grad == 2).all()
    g, beta = inner.inner.gates(torch.full((2, 3, 5), 0.01, dtype=dtype))
    assert g.dtype == beta.dtype == torch.float32 and (g < 0).all()
