"""The rows and weights of mxfp4_exact.py without a GPU: their products are exact in f32, and
every output set changes when a term or digit of the rows is lost."""
import numpy as np
import pytest

import mxfp4 as mx
from mxfp4_choice import BF16, F16, F32, MANY, PLANES
from mxfp4_exact import dense_rows, dense_weights, digits, exponents, sparse_rows, sparse_weights, terms

CASES = sorted({(v[0], c[0], c[2], min(c[3], 64)) for c, v in MANY.items()})


def sets(rng, t, k, rows, pair):
    e = exponents(rng, t, rows, pair)
    yield dense_rows(rng, t, rows, k, e), mx.values(*dense_weights(rng, 8, k))
    if t != PLANES:
        yield sparse_rows(rng, t, rows, k, e), mx.values(*sparse_weights(rng, 8, k))


@pytest.mark.parametrize("kind,t,k,rows,pair", [(*c, p) for c in CASES for p in (False, True) if not p or c[1] in (F32, PLANES)])
def test_products_are_exact(kind, t, k, rows, pair):
    """Sums in f32, forwards and backwards, give the float64 result; so do those of the parts."""
    rng = np.random.default_rng(k + t)
    for (_, x), w in sets(rng, t, k, rows, pair):
        parts = digits(x) if kind == "digits" else [x] if t == PLANES else terms(x, 3 if t == F32 else 2 if t == F16 else 1)
        assert np.array_equal(sum(parts), x)
        want = x @ w.T
        for order in (parts, parts[::-1]):
            y = np.zeros(want.shape, np.float32)
            for i in range(k):
                for p in order:
                    y += (p[:, i:i + 1] * w[:, i]).astype(np.float32)
            assert np.array_equal(y, want)


@pytest.mark.parametrize("kind,t,k,rows", [c for c in CASES if c[0] != "planes" and c[1] != BF16])
def test_every_part_counts(kind, t, k, rows):
    """Without any one of its parts, at least one output in ten of a set is off by 2^-18 of
    itself (the tolerance of a pair is 2^-20)."""
    rng = np.random.default_rng(k + t)
    seen = None
    for (_, x), w in sets(rng, t, k, rows, False):
        parts = digits(x) if kind == "digits" else terms(x, 3 if t == F32 else 2)
        want = x @ w.T
        off = [np.mean(np.abs((x - p) @ w.T - want) > 2.0 ** -18 * np.abs(want)) for p in parts]
        seen = off if seen is None else np.maximum(seen, off)
    assert min(seen) > 0.1, seen
