"""The list of tests/linear_shapes.py against the library's answers (no GPU): each size takes the kernel it stands for, and no size takes one that the
list has not.  A constant of the plan that moves fails here, with the size that has to be found again."""
import random

import pytest

from tests.linear_shapes import BF16, F32, FWD, GW, GX, ROWS, SHAPES, STAGED, STREAM, linear_kernel


@pytest.mark.parametrize("key", SHAPES, ids=str)
def test_sizes_take_their_kernel(key):
    dtype, product, family, shape, shared = key
    got = linear_kernel(*SHAPES[key], product, dtype, family == STREAM)
    assert got[:2] == (family, shape) and (got[2] > 1) == shared


def test_no_size_takes_another_kernel():
    have = {key[:4] for key in SHAPES}
    assert {(d, p, s) for d, p, f, s in have if f == STREAM} == {(BF16, p, s) for p in (FWD, GX, GW) for s in range(4)}
    assert {(d, p, s) for d, p, f, s in have if f == STAGED} == {(d, p, s) for d in (F32, BF16) for p in (FWD, GX, GW) for s in range(4 if d == F32 else 2)}
    assert {(d, p, s) for d, p, f, s in have if f == ROWS} == {(d, FWD, s) for d in (F32, BF16) for s in (1, 2, 4)}
    r = random.Random(7)
    for _ in range(20000):
        rows, k, n = (int(2 ** r.uniform(0, 15)) for _ in range(3))
        for dtype in (F32, BF16):
            for product in (FWD, GX, GW):
                for aligned in (False, True):
                    for outputs in (1, 2) if product == FWD else (1,):
                        got = linear_kernel(rows, k, n, product, dtype, aligned, outputs)
                        assert (dtype, product, got[0], got[1]) in have, (rows, k, n)


def test_the_query_refuses():
    import ctypes
    from addernetcuda_amd._lib import lib
    ask = lambda rows=8, k=8, n=8, product=0, dtype=0, outputs=1: lib.adder_linear_kernel(rows, k, n, product, dtype, 1, outputs, ctypes.byref(ctypes.c_int()))
    assert ask() == 0 and ask(outputs=2) == 0
    for bad in ({"rows": 0}, {"n": -1}, {"product": 3}, {"product": -1}, {"dtype": 2}, {"outputs": 0}, {"outputs": 3}, {"product": 1, "outputs": 2}):
        assert ask(**bad) == -2, bad
    assert ask(rows=1 << 40) == -3 and lib.adder_linear_kernel(8, 8, 8, 0, 0, 1, 1, None) == -1
