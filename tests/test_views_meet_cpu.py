"""Whether two views share memory (the refusals of outputs that lie over what a call reads), against the sets of their elements."""
import ctypes

import numpy as np
import pytest

from kandle_b200 import lib

BF16, F32 = lib.DTYPES["bfloat16"][0], lib.DTYPES["float32"][0]


def view(shape, strides, offset=0, dtype=BF16, storage=1):
    t = lib.kd_tensor()
    t.storage, t.offset, t.dtype, t.ndim = storage, offset, dtype, len(shape)
    for i, (n, s) in enumerate(zip(shape, strides)):
        t.shape[i], t.strides[i] = n, s
    return t


def meet(a, b):
    out = ctypes.c_int(-1)
    lib.call("kd_debug_views_meet", ctypes.byref(a), ctypes.byref(b), ctypes.byref(out))
    return bool(out.value)


def elements(t):
    at = np.zeros(1, np.int64) + t.offset
    for i in range(t.ndim):
        at = (at[:, None] + np.arange(t.shape[i]) * t.strides[i]).reshape(-1)
    return set(at.tolist())


def test_heads_of_one_buffer():
    """[tokens, heads, 64] views of a [tokens, 24 * 64] buffer: apart, in turn, and over one another by one element."""
    row = 24 * 64
    q = view((100, 8, 64), (row, 64, 1))
    assert not meet(q, view((100, 8, 64), (row, 64, 1), 8 * 64)) and not meet(view((100, 8, 64), (row, 64, 1), 16 * 64), q)
    assert meet(q, view((100, 8, 64), (row, 64, 1), 7 * 64)) and meet(q, view((100, 8, 64), (row, 64, 1), 8 * 64 - 1))
    even, odd = view((100, 8, 64), (row, 128, 1)), view((100, 8, 64), (row, 128, 1), 64)
    assert not meet(even, odd) and meet(even, even) and meet(even, view((100, 8, 64), (row, 128, 1), 63))
    assert meet(q, view((100, 8, 64), (row, 64, 1), row)) and not meet(q, view((100, 8, 64), (row, 64, 1), 100 * row))
    assert meet(q, view((99, 8, 64), (row, 64, 1), row + 8)) and not meet(q, view((1, 8, 64), (7, 64, 1), 98 * row + 8 * 64))


def test_spans_decide_where_the_layouts_differ():
    a = view((4, 8), (8, 1))
    assert not meet(a, view((2, 8), (1, 2), 32)) and meet(a, view((2, 8), (1, 2), 31)) and meet(a, view((8,), (1,), 3))
    assert meet(a, view((4,), (1,), 15, F32)) and not meet(a, view((4,), (1,), 16, F32))
    assert not meet(a, view((4, 8), (8, 1), storage=2)) and not meet(a, view((0, 8), (8, 1))) and not meet(view((3, 0), (1, 1)), a)


@pytest.mark.parametrize("seed", range(4))
def test_views_of_equal_strides_against_their_elements(seed):
    rng = np.random.default_rng(seed)
    both = [0, 0]
    for _ in range(1500):
        dims = int(rng.integers(1, 4))
        inner, strides = 1, []
        for _ in range(dims):                       # nested, with gaps, in any order, some the other way round
            strides.append(inner * int(rng.integers(1, 4)) * (1 if rng.random() < 0.8 else -1))
            inner = abs(strides[-1]) * int(rng.integers(1, 6))
        order = rng.permutation(dims)
        strides = [strides[i] for i in order]
        shapes = [[int(rng.integers(1, 6)) for _ in range(dims)] for _ in range(2)]
        a = view(shapes[0], strides, 500)
        b = view(shapes[1], [s if n > 1 or rng.random() < 0.5 else 9 for s, n in zip(strides, shapes[1])], 500 + int(rng.integers(-40, 41)))
        want = bool(elements(a) & elements(b))
        assert meet(a, b) == want == meet(b, a)
        both[want] += 1
    assert min(both) > 200


def bytes_of(t):
    size = {F32: 4, BF16: 2}[t.dtype]
    return {e * size + i for e in elements(t) for i in range(size)}


def test_a_small_view_in_the_gaps_of_another():
    """A row's padding holds something else: one number, a short list, of another type or rank."""
    table = view((50, 6), (10, 1), 0, F32)
    for at in (6, 9, 26, 496):
        assert not meet(table, view((1,), (1,), at, F32)) and not meet(view((1, 2), (2, 1), at - at % 10 + 6, F32), table)
    assert meet(table, view((1,), (1,), 25, F32)) and meet(table, view((2,), (1,), 9, F32)) and not meet(table, view((40,), (10,), 7, F32))
    assert not meet(table, view((8,), (1,), 12)) and meet(table, view((9,), (1,), 12)) and not meet(view((2, 3), (20, 1), 13), table)
    assert meet(view((70, 80), (200, 2)), view((80, 70), (2, 201), 1)), "large and unlike: the spans decide"


@pytest.mark.parametrize("seed", range(4))
def test_small_views_of_any_strides_against_their_bytes(seed):
    rng = np.random.default_rng(seed)
    both = [0, 0]
    for _ in range(1500):
        pair = []
        for _ in range(2):
            dims, inner, strides, shape = int(rng.integers(1, 4)), 1, [], []
            for _ in range(dims):
                strides.append(inner * int(rng.integers(1, 4)) * (1 if rng.random() < 0.8 else -1))
                shape.append(int(rng.integers(1, 5)))
                inner = abs(strides[-1]) * int(rng.integers(1, 6))
            dtype = F32 if rng.random() < 0.5 else BF16
            pair.append(view(shape, strides, (250 if dtype == F32 else 500) + int(rng.integers(-30, 31)), dtype))
        a, b = pair
        want = bool(bytes_of(a) & bytes_of(b))
        assert meet(a, b) == want == meet(b, a)
        both[want] += 1
    assert min(both) > 200
