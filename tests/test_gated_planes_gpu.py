"""Float32 results of the gated recurrence as a whole, against float64: their operands keep three planes of bf16.

Bounds, of a result's norm.  Three planes keep 24 bits.  The tensor cores truncate as they add: a third of 2^-23 of the accumulator on
average (half a last place of 24 bits, which is between 2^-24 and 2^-23 of the value).  A product over 64 terms is four steps of 16,
whose accumulator grows with the root of its terms: of half, 0.71, 0.87 and all of the result, 3.1 in sum.
  bf16 inputs, one operand in three planes: three additions a step, 3.1 * 2^-23 a product.  State and its gradient are one product,
  gradients of gates two behind one another: 6.2 * 2^-23, below 2^-20.
  float32 inputs, six pairs of planes: 6.2 * 2^-23 a product, two behind one another 12.4 * 2^-23, below 2^-19.
With two planes a factor is off by 2.5e-6 = 2^-18.6 on average (`test_two_planes_do_not_meet_the_bounds`), above both.  The element by
element bounds of the other tests, of the worst case, do not tell two planes from three."""

import pytest
import torch

import test_gated_linear_gpu as G
from oracle import gated_oracle as O

BF16_BOUND, F32_BOUND = 2.0 ** -20, 2.0 ** -19
# one block per stream, segments, and ranges of streams (forward and backward; backward alone)
SHAPES = [(2, 3, 200, 64), (2, 3, 200, 32), (1, 1, 1300, 64), (45, 10, 70, 64), (30, 10, 130, 32)]


def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,T,F", SHAPES)
def test_float32_results_keep_their_digits(B, H, T, F, dtype):
    ins, d_out, d_w = G.make(B, H, T, F, dtype, seed=T + F)
    got = G.run(ins, d_out, d_w)
    with torch.device("cuda"):
        want = O.gated_grads(*[t.cuda() for t in G.f64(ins)], d_out.cuda().double(), d_w.cuda().double())
    for name, x, y in zip(G.NAMES, got, want):
        if dtype == torch.bfloat16 and name in G.BF16:
            continue
        assert off(x, y) <= (BF16_BOUND if dtype == torch.bfloat16 else F32_BOUND), (name, off(x, y))
    forward = G.run(ins)
    assert off(forward[1], want[1]) <= (BF16_BOUND if dtype == torch.bfloat16 else F32_BOUND)
    if dtype == torch.float32:
        assert off(forward[0], want[0]) <= F32_BOUND


def planes(x, n):
    """x [float32 values in float64] as the sum of n bf16 planes."""
    y = torch.zeros_like(x)
    for _ in range(n):
        y = y + (x - y).bfloat16().double()
    return y


@pytest.mark.parametrize("n", [2, 3])
def test_two_planes_do_not_meet_the_bounds(n):
    """A state of 64 tokens, its scaled keys in n planes (bf16 inputs); keys and values in n planes (float32 inputs)."""
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(64, 64, generator=g).double() for _ in range(2))
    scale = torch.rand(64, 1, generator=g).double()
    b = [t.bfloat16().double() for t in (k, v)]
    keys = (b[0] * scale).float().double()
    bf16, f32 = off(planes(keys, n).T @ b[1], keys.T @ b[1]), off(planes(k, n).T @ planes(v, n), k.T @ v)
    one = off(planes(k, n).T @ v, k.T @ v)
    assert (bf16 > 2 * BF16_BOUND and f32 > 1.5 * F32_BOUND and one > F32_BOUND) if n == 2 else max(bf16, f32) < 2.0 ** -24
