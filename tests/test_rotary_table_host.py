"""CPU-only checks of a rotation's table: how long it lives, and what it may be used for."""

import torch

import ttt_rs_b200 as tb


def test_a_table_made_in_inference_mode_is_an_ordinary_tensor():
    """Autograd does not save inference tensors: a rotation made while serving could not be differentiated later."""
    with torch.inference_mode():
        rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cpu")
    assert not rot.turns.is_inference() and rot._args[0] is rot.turns
    assert torch.equal(rot.turns, tb.Rotary(tb.RotaryConfig(head_dim=64), device="cpu").turns)
