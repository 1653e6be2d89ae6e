"""Which results of the rotary operators lie over another tensor: the decision against sets of addresses, and the refusals."""

import ctypes as C
import itertools
import random

import pytest

from ttt_rs_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from ttt_rs_b200.build import build
    build()
    return _lib.load()


def ints(x):
    return C.cast((C.c_int64 * len(x))(*x), C.c_void_p)


def meet(lib, F, a, b, es=2, base=0x10000):
    """a, b: (first element, sizes, strides)"""
    return bool(lib.ttt_internal_rows_meet(F, es, C.c_void_p(base + es * a[0]), ints(a[1]), ints(a[2]), C.c_void_p(base + es * b[0]),
                                           ints(b[1]), ints(b[2])))


def elements(F, t):
    at, sizes, strides = t
    return {at + sum(i * s for i, s in zip(idx, strides)) + f for idx in itertools.product(*map(range, sizes)) for f in range(F)}


def view(rng, F):
    """Sizes and strides of a tensor as they come: dense, turned, columns of a projection, a padded cache, or anything."""
    B, H, T = (rng.choice((1, 1, 2, 3)) for _ in range(3))
    kind = rng.randrange(5)
    if kind == 0:
        strides = (H * T * F, T * F, F)
    elif kind == 1:
        strides = (H * T * F, F, H * F)
    elif kind == 2:
        pitch = H * F + rng.choice((0, F, 2 * F, 3))
        strides = (T * pitch, F, pitch)
    elif kind == 3:
        most = T + rng.choice((0, 1, 2))
        strides = (H * most * F, most * F, F)
    else:
        strides = tuple(rng.randrange(0, 3 * F) for _ in range(3))
    return (B, H, T), tuple(0 if n == 1 else s for n, s in zip((B, H, T), strides))


def test_the_decision_is_that_of_the_addresses(lib):
    rng = random.Random(4)
    seen = [0, 0]
    for _ in range(20000):
        F = rng.choice((2, 4, 6))
        a, b = view(rng, F), view(rng, F)
        if rng.random() < 0.5:  # (two blocks of one layout)
            b = a
        at = rng.randrange(0, 60), rng.randrange(0, 60)
        x, y = (at[0], *a), (at[1], *b)
        want = bool(elements(F, x) & elements(F, y))
        seen[want] += 1
        assert meet(lib, F, x, y, es=rng.choice((2, 4))) == want, (F, x, y)
    assert min(seen) > 4000


def test_views_of_a_projection_and_of_a_cache(lib):
    B, H, T, F, pitch = 2, 3, 500, 64, 4 * 3 * 64 + 8
    cols = lambda at, heads=H: (at, (B, heads, T), (T * pitch, F, pitch))  # noqa: E731
    assert not meet(lib, F, cols(0), cols(H * F)) and not meet(lib, F, cols(H * F, 1), cols(0)) and not meet(lib, F, cols(0), cols(pitch - H * F))
    assert meet(lib, F, cols(0), cols(H * F - 2)) and meet(lib, F, cols(H * F), cols(2)) and meet(lib, F, cols(0), cols(pitch))
    each_other = lambda at: (at, (B, H, T), (T * pitch, 2 * F, pitch))  # noqa: E731  (queries and keys head by head)
    assert not meet(lib, F, each_other(0), each_other(F)) and meet(lib, F, each_other(0), each_other(F - 1))
    cache = lambda t: (t * F, (B, H, T), (H * (T + 9) * F, (T + 9) * F, F))  # noqa: E731
    assert meet(lib, F, cache(0), cache(1)) and meet(lib, F, cache(9), cache(0))
    tail = (T * F, (B, H, 9), (H * (T + 9) * F, (T + 9) * F, F))
    assert not meet(lib, F, cache(0), tail) and not meet(lib, F, tail, cache(0))
    # what would be behind 32 and 63 bits
    far = lambda at: (at, (1 << 20, 1 << 10, 1 << 20), (1 << 42, 1 << 32, 1 << 8))  # noqa: E731
    assert not meet(lib, F, far(0), far(64)) and meet(lib, F, far(0), far(63))


def test_results_over_another_tensor_are_refused(lib):
    """Nothing is launched: every call is refused."""
    es, F, T, pitch = 2, 64, 10, 3 * 3 * 64
    d = _lib.TttDims(2, 3, T, F, 0, 0, 1e-6, 1)
    rot = _lib.TttRotation(0x1000, None, 0, 0, 64, 0, 0, 1.0)
    at = lambda e: C.c_void_p(0x100000 + es * e)  # noqa: E731
    cols = [T * pitch, F, pitch]

    def rotary(x, y, s):
        return lib.ttt_layer_rotary(C.byref(d), at(x), ints(s), C.byref(rot), 0, at(y), ints(s), None)

    def norm(q, k, yq, yk, s=cols):
        return lib.ttt_layer_qk_norm_rotary(C.byref(d), 3, at(q), at(k), ints(s * 2), None, None, C.byref(rot), at(yq), at(yk), ints(s * 2), None)

    cache = [3 * (T + 2) * F, (T + 2) * F, F]
    assert rotary(0, F, cache) == rotary(0, 8, cols) == rotary(8, 0, cols) == _lib.TTT_ERR_SHAPE
    assert "lies over" in _lib.last_error()
    block = 3 * F
    assert norm(0, block, block, 0) == norm(0, block, 0, 0) == norm(0, block, 0, 8) == norm(0, block, 2 * block, block - 8) == _lib.TTT_ERR_SHAPE
    need = lib.ttt_layer_qk_norm_rotary_backward_workspace_bytes(C.byref(d), 3)

    def backward(q, k, gq, gk, dq, dk):
        return lib.ttt_layer_qk_norm_rotary_backward(C.byref(d), 3, at(q), at(k), at(gq), at(gk), ints(cols * 4), None, None, C.byref(rot),
                                                     at(dq), at(dk), ints(cols * 2), C.c_void_p(0x1000), None, C.c_void_p(0x1000), need, None)

    far = 1 << 20
    assert backward(0, block, far, far + block, far + block, 2 * far) == backward(0, block, far, far + block, 8, 2 * far) == _lib.TTT_ERR_SHAPE
    assert backward(0, block, far, far + block, 2 * far, 2 * far) == backward(0, block, far, far + block, 2 * far, 0) == _lib.TTT_ERR_SHAPE
