"""CPU-only checks of layers whose queries and keys are normed or rotated otherwise, and of those that are not."""

import pytest
import torch

import ttt_rs_b200 as tb


@pytest.mark.parametrize("kw", [dict(rope_theta=0.5), dict(rope_theta=0.5, pos_encoding="rope_global"), dict(hidden_size=126),
                                dict(hidden_size=1024), dict(pos_encoding="none", rope_theta=0.0)])
def test_layers_without_heads_of_their_own_are_built_as_before(kw):
    """The limits of the rotary operators (theta of at least 1, even heads up to 256) are theirs alone."""
    cfg = tb.TTTLayerConfig(**{**dict(hidden_size=128, num_heads=2), **kw})
    assert not cfg.own_heads
    assert tb.TTT(cfg).q_norm_weight is None


@pytest.mark.parametrize("kw", [dict(rope_theta=0.5), dict(hidden_size=126), dict(hidden_size=1024)])
@pytest.mark.parametrize("own", [dict(qk_norm=True), dict(rope_layout="half")])
def test_heads_of_their_own_have_the_operators_limits(kw, own):
    with pytest.raises(ValueError):
        tb.TTT(tb.TTTLayerConfig(**{**dict(hidden_size=128, num_heads=2), **kw, **own}))


def test_own_heads():
    own = lambda **kw: tb.TTTLayerConfig(128, 2, **kw).own_heads  # noqa: E731
    assert not own() and not own(rotary_dim=64) and not own(pos_encoding="none", rope_layout="half") and not own(rope_factor=4.0)
    assert own(qk_norm=True) and own(qk_norm=True, pos_encoding="none")
    assert own(rotary_dim=32) and own(rope_layout="half") and own(rope_scaling="linear", rope_factor=2.0)
