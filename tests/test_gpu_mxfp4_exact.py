"""MXFP4 products at sizes that take each form of the kernels (asserted), on rows and weights
whose products are exact in f32 (mxfp4_exact.py): outputs bit for bit."""
import numpy as np
import pytest

import mxfp4 as mx
from mxfp4_choice import FEW, MANY, PLANES, taken
from mxfp4_exact import dense_rows, dense_weights, exponents, sparse_rows, sparse_weights
from test_gpu_mxfp4 import buf, matrix, run_planes, run_rows  # noqa: F401

pytestmark = pytest.mark.gpu


def check(dev, buf, case, weights, rows_of):
    t, n, k, rows, pair = case
    rng = np.random.default_rng(n + k + rows)
    w, u = weights(rng, n, k), weights(rng, n, k) if pair else None
    raw, x = rows_of(rng, t, rows, k, exponents(rng, t, rows, pair))
    m, up = matrix(dev, w), matrix(dev, u) if pair else None
    run = (lambda **a: run_planes(dev, buf, m, raw, up=up, **a)) if t == PLANES else \
        (lambda **a: run_rows(dev, buf, m, raw, t, up=up, **a))
    y = x @ mx.values(*w).T
    got = run(ldy_more=rows % 2)
    if pair:
        # the epilogue's exp, division and product: under 8 roundings of 2^-23. A gate below
        # -88.72 has exp(-g) past the largest f32, 2^128, and silu(g) as -0: off by 88.73 exp(-88.72)
        # < 2^6.5 2^-127.9 at most, times the up product
        with np.errstate(over="ignore"):
            up_y = x @ mx.values(*u).T
            want = mx.silu(y) * up_y
        assert (np.abs(got - want) <= 2.0 ** -20 * np.abs(want) + 2.0 ** -121 * np.abs(up_y) + 2.0 ** -126).all()
        return
    assert np.array_equal(got, y)
    # a residual that keeps the sum a number of f32: the negative of the product's half
    res = (-y / 2).astype(np.float32)
    assert np.array_equal(run(res=res, ldy_more=3), y / 2)


@pytest.mark.parametrize("case", [*MANY, *FEW])
def test_whole_numbers(dev, buf, case):
    assert case not in MANY or taken(*case) == MANY[case]
    check(dev, buf, case, dense_weights, dense_rows)


@pytest.mark.parametrize("case", [c for c in [*MANY, *FEW] if c[0] != PLANES])
def test_all_bits_of_a_value(dev, buf, case):
    assert case not in MANY or taken(*case) == MANY[case]
    check(dev, buf, case, sparse_weights, sparse_rows)
