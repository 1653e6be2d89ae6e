"""Norm and rotation at sizes where the gradient's blocks take several tokens each and the forward's several rounds: float32, and rows
that are read feature by feature.  Bounds as in test_rotary_gpu.py."""

import pytest
import torch

import test_rotary_gpu as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("F,rdim,layout", [(64, None, "tokens"), (80, 20, "tokens"), (64, None, "odd"), (256, None, "heads"), (130, 66, "heads")])
def test_norm_of_many_rows(F, rdim, layout, dtype):
    import ttt_rs_b200 as tb
    for pairs in ("interleaved", "half"):
        R.check_qk(tb.RotaryConfig(head_dim=F, rotary_dim=rdim, layout=pairs), 3, 6, 2, 2999, F, dtype, layout=layout)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("F,rdim,layout", [(80, 20, "tokens"), (64, None, "odd"), (256, 250, "heads"), (32, None, "tokens")])
def test_rotation_of_many_rows(F, rdim, layout, dtype):
    import ttt_rs_b200 as tb
    for pairs in ("interleaved", "half"):
        R.check_rotary(tb.RotaryConfig(head_dim=F, rotary_dim=rdim, layout=pairs), 3, 5, 8001, dtype, layout=layout)
