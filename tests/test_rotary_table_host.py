"""CPU-only checks of a rotation's table: how long it lives, and what it may be used for."""

import torch

import ttt_rs_b200 as tb


def test_a_table_made_in_inference_mode_is_an_ordinary_tensor():
    """Autograd does not save inference tensors: a rotation made while serving could not be differentiated later."""
    with torch.inference_mode():
        rot = tb.Rotary(tb.RotaryConfig(head_dim=64), device="cpu")
    assert not rot.turns.is_inference() and rot._args[0] is rot.turns
    assert torch.equal(rot.turns, tb.Rotary(tb.RotaryConfig(head_dim=64), device="cpu").turns)


def test_a_layers_table_stays_where_captured_graphs_read_it():
    """However many other configurations come after it (a table is a kilobyte at most)."""
    from ttt_rs_b200.layer import _layer_rotary
    cfgs = [tb.TTTLayerConfig(128, 2, rope_layout="half", rope_theta=1000.0 + i) for i in range(200)]
    cpu = torch.device("cpu")
    first = _layer_rotary(cfgs[0], cpu)
    for c in cfgs:
        _layer_rotary(c, cpu)
    assert _layer_rotary(cfgs[0], cpu) is first
