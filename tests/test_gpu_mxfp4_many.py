"""MXFP4 products of special values at sizes that take the many-row kernel (asserted):
rounding of f32 rows held in digits, infinities and NaN, NaN blocks of weights."""
import numpy as np
import pytest

import mxfp4 as mx
from mxfp4_choice import BF16, F16, F32, MANY, PLANES, choice, taken
from test_gpu_mxfp4 import buf, matrix, run_planes, run_rows, weights  # noqa: F401
from test_gpu_mxfp4_launches import Graph, big, fill, put  # noqa: F401

pytestmark = pytest.mark.gpu


def sizes(want):
    """The sizes of MANY whose entry passes."""
    return [c for c, v in MANY.items() if want(c, v)]


def product(dev, buf, m, t, raw, up=None):
    return run_planes(dev, buf, m, raw, up=up) if t == PLANES else run_rows(dev, buf, m, raw, t, up=up)


@pytest.mark.parametrize("case", sizes(lambda c, v: v[0] == "digits" and not c[4]))
def test_digits_round_to_their_step(dev, buf, case):
    """One value a row whose weights are not zero, 2^8 to 2^29 below its block's largest,
    1.5 2^e: rows are held within 2^-30 of the power of two above that one, and the product with
    a weight of 2 bits is exact in f32, so outputs are off by 2^(e + 1 - 30) times the weight at
    most. (30 bits with the sign: |x| < 2^(e + 1) as whole numbers up to 2^29 makes steps of
    2^(e - 28), half of one 2^(e - 29). Three digits less are 2^15 times as far off.)"""
    assert taken(*case) == MANY[case]
    t, n, k, rows, _ = case
    rng = np.random.default_rng(n + k)
    codes, scales = weights(rng, n, k)
    codes[:, 0::16] &= 0xF0  # each block's first element
    wv = mx.values(codes, scales)
    r = np.arange(rows)
    col = rng.integers(0, k // 32, rows) * 32 + rng.integers(1, 32, rows)
    e = rng.integers(-30, 30, rows)
    x = np.zeros((rows, k), np.float32)
    x[r, col // 32 * 32] = 1.5 * 2.0 ** e
    x[r, col] = rng.uniform(-2, 2, rows) * 2.0 ** (e - rng.integers(8, 30, rows))
    want = x[r, col].astype(np.float64)[:, None] * wv[:, col].T
    got = run_rows(dev, buf, matrix(dev, (codes, scales)), x, t)
    assert (np.abs(got - want) <= 2.0 ** (e - 29.0)[:, None] * np.abs(wv[:, col].T)).all()


@pytest.mark.parametrize("case", sizes(lambda c, v: True))
def test_nonfinite_stays_in_its_row_and_column(dev, buf, case):
    """A NaN in a row's first block, an infinity in another's last and a NaN block of weights:
    NaN for the first (and for f32 rows in digits the second), an infinity by the weight's sign
    (NaN where the weight is zero) for the second otherwise, NaN in the weights' column. All
    other outputs keep the bits that they have when the bad values are ordinary ones."""
    assert taken(*case) == MANY[case]
    t, n, k, rows, pair = case
    rng = np.random.default_rng(n + k + rows)
    w, u = weights(rng, n, k), weights(rng, n, k) if pair else None
    w[1][n - 5, k // 32 - 1] = 255  # in the last k tile
    wv = mx.values(*w)
    m, up = matrix(dev, w), matrix(dev, u) if pair else None
    nan_row, inf_row = rows // 2, rows - 1
    if t == PLANES:
        raw = weights(rng, rows, k, spread=5)
        good = product(dev, buf, m, t, raw, up)
        raw[1][nan_row, 0] = raw[1][inf_row, k // 32 - 1] = 255
    else:
        x = rng.normal(0, 1, (rows, k)).astype(np.float32)
        raw, _ = mx.rows_of(x, t)
        good = product(dev, buf, m, t, raw, up)
        raw = raw.copy()
        raw[nan_row, 3] = 0x7FC0 if t == BF16 else np.nan
        raw[inf_row, k - 1] = 0x7F80 if t == BF16 else np.inf
    got = product(dev, buf, m, t, raw, up)
    assert np.isnan(good[:, n - 5]).all() and np.isnan(got[:, n - 5]).all()
    live = np.arange(n) != n - 5
    assert np.isfinite(good[:, live]).all()
    assert np.isnan(got[nan_row]).all()
    if t == PLANES or MANY[case][0] == "digits":
        assert np.isnan(got[inf_row]).all()
    elif not pair:
        with np.errstate(invalid="ignore"):
            assert np.array_equal(got[inf_row, live], (np.inf * wv[:, k - 1])[live], equal_nan=True)
    else:  # (silu of minus infinity is NaN, as are products of infinities with zeros)
        assert not np.isfinite(got[inf_row]).any()
    rest = np.ones(rows, bool)
    rest[[nan_row, inf_row]] = False
    assert np.array_equal(got[rest][:, live].view(np.uint32), good[rest][:, live].view(np.uint32))


DIGITS = sizes(lambda c, v: v[0] == "digits" and not c[4])


@pytest.mark.parametrize("case", DIGITS)
def test_digits_near_the_largest_number(dev, buf, case):
    """Products just below 2^128, exact in f32: no leading digits of a value, rounded up, may
    carry a sum past it. Rows in turn: a value of all ones (the digits of its leading half are
    2^128 with the weight); the same far below the largest f32, under large weights; three
    values beside an outlier whose top digit is 1.9375 times each; negated."""
    assert taken(*case) == MANY[case]
    t, n, k, rows, _ = case
    rng = np.random.default_rng(n + k)
    # each block: a zero weight, then ones of the output's sign; scales 1, 2^20 and 8 in turn
    sign = rng.integers(0, 2, n).astype(np.uint8) * 0x88
    codes = np.tile((0x22 | sign)[:, None], (1, k // 2)).astype(np.uint8)
    codes[:, 0::16] &= 0xF0
    scales = np.tile(np.resize(np.array([127, 147, 130], np.uint8), k // 32), (n, 1))
    x = np.zeros((rows, k), np.float32)
    r = np.arange(rows)
    block = rng.integers(0, k // 96, rows) * 3 + r % 3
    big = 2.0 ** 128 - 2.0 ** 104  # the largest f32
    col = block * 32 + rng.integers(1, 28, rows)
    x[r, col] = np.where(r % 3 == 1, big * 2.0 ** -20, big)
    far = r[r % 3 == 2]
    x[far, col[far]] = 0
    x[far, block[far] * 32] = 2.0 ** 127  # steps of 2^99
    for i in range(3):  # in those steps 32^5 / 1.9375, so a top digit of 1: 2^124, times 8 and thrice
        x[far, col[far] + i] = float.fromhex("0x1084212p99")
    x[r % 2 == 1] *= -1
    w = mx.values(codes, scales)
    want = x.astype(np.float64) @ w.T
    assert np.abs(want).max() < 2.0 ** 128 and (np.abs(want) > 2.0 ** 127).all()
    got = run_rows(dev, buf, matrix(dev, (codes, scales)), x, t)
    # (three values: two additions of numbers below 2^128, each at most 2^-23 of the sum off, per digit)
    assert (np.abs(got - want) <= 12 * 2.0 ** -23 * np.abs(want)).all()
    one = r % 3 < 2
    assert np.array_equal(got[one], want[one])


@pytest.mark.parametrize("case", DIGITS)
def test_results_past_the_largest_number(dev, buf, case):
    """Never a finite number: an infinity, or a NaN where the digits' products pass it with both
    signs. The other rows keep their bits."""
    assert taken(*case) == MANY[case]
    t, n, k, rows, _ = case
    rng = np.random.default_rng(n + k)
    w = np.where(rng.random((n, k // 2)) < 0.5, 0x66, 0xEE).astype(np.uint8), np.full((n, k // 32), 127, np.uint8)  # +-4
    m = matrix(dev, w)
    x = rng.normal(0, 1, (rows, k)).astype(np.float32)
    good = run_rows(dev, buf, m, x, t)
    past = np.arange(0, rows, 3)
    x[past] = 0
    x[past, rng.integers(0, k, past.size)] = rng.uniform(1, 2, past.size) * 2.0 ** rng.integers(126, 128, past.size)
    got = run_rows(dev, buf, m, x, t)
    assert not np.isfinite(got[past]).any()
    rest = np.arange(rows) % 3 > 0
    assert np.array_equal(got[rest].view(np.uint32), good[rest].view(np.uint32))


@pytest.mark.parametrize("case", DIGITS)
def test_digits_below_the_normal_range(dev, buf, case):
    """One value a row, 2^-140 to 2^-95, under weights of 2^100 times their codes: blocks below
    2^-100 are held in steps of 2^-129. Then large values under weights of the smallest scale,
    whose products are exact."""
    assert taken(*case) == MANY[case]
    t, n, k, rows, _ = case
    rng = np.random.default_rng(n + k)
    r, col = np.arange(rows), rng.integers(0, k, rows)
    x = np.zeros((rows, k), np.float32)
    x[r, col] = rng.uniform(-2, 2, rows) * 2.0 ** rng.integers(-140, -95, rows)
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    w = codes, np.full((n, k // 32), 227, np.uint8)
    wv = mx.values(*w)[:, col].T
    want = x[r, col].astype(np.float64)[:, None] * wv
    got = run_rows(dev, buf, matrix(dev, w), x, t)
    # (five additions of digits of up to 24 bits)
    assert (np.abs(got - want) <= 2.0 ** -130 * np.abs(wv) + 10 * 2.0 ** -23 * np.abs(want)).all()
    x = np.where(x != 0, np.float32(1.25 * 2.0 ** 100), np.float32(0))
    w = codes, np.zeros((n, k // 32), np.uint8)
    want = x[r, col].astype(np.float64)[:, None] * mx.values(*w)[:, col].T
    assert np.array_equal(run_rows(dev, buf, matrix(dev, w), x, t), want)


@pytest.mark.parametrize("t", [F32, PLANES])
@pytest.mark.parametrize("n,pair", [((1 << 28) + 77, True), ((1 << 29) + 77, False)])
def test_outputs_past_one_launch(big, t, n, pair):
    """Row tiles of a matrix that need more workgroups of the few-row kernel than a grid
    holds (one or two of them each): most weights are zeros, the others lie at both ends and
    around the place where the second launch begins."""
    from pagoda_amd import Matrix

    dev, buf = big
    rng = np.random.default_rng(n + t)
    k, rows, ld = 32, 2, 16
    assert not choice(t, n, k, rows, pair).block
    pc, ps, py = dev.alloc(n * ld), dev.alloc(n * ld), dev.alloc(rows * n * 4)
    buf.ptrs += [pc, ps, py]
    fill(dev, pc, 0, n * ld)
    fill(dev, ps, 127, n * ld)
    cut = ((1 << 24) - 64) * (1 if pair else 2) * 16
    ws = []
    for r0 in (0, cut - 100, n - 200):
        codes, _ = weights(rng, 200, k)
        ws.append((r0, codes))
        put(dev, pc + r0 * ld, codes)
    m = Matrix.from_mxfp4_dev(dev, pc, ld, ps, ld, n, k)
    if t == PLANES:
        raw = weights(rng, rows, k)
        x = mx.values(*raw)
        xs = buf.up(mx.padded(raw[0], ld, np.uint8(0))), ld, buf.up(mx.padded(raw[1], ld, np.uint8(0))), ld
        if pair:
            Matrix.gemv_swiglu_mx_dev(m, m, *xs, rows, py, n)
        else:
            m.gemv_mx_dev(*xs, rows, py, n)
    else:
        x = rng.normal(0, 1, (rows, k)).astype(np.float32)
        px = buf.up(x)
        x = x.astype(np.float64)
        if pair:
            Matrix.gemv_swiglu_dev(m, m, px, k, rows, py, n)
        else:
            m.gemv_dev(px, k, rows, py, n)
    for r in range(rows):
        for r0, codes in ws:
            at = max(r0 - 100, 0)
            got = dev.download(py + (r * n + at) * 4, (min(500, n - at),), np.float32)
            live = got[r0 - at:r0 - at + 200]
            wv = mx.values(codes, np.full((200, 1), 127, np.uint8))
            y, xr = x[r] @ wv.T, x[r:r + 1]
            if pair:
                assert (np.abs(live - mx.silu(y) * y) <= mx.swiglu_bound(xr, wv, wv)[0]).all()
            else:
                assert (np.abs(live - y) <= mx.product_bound(xr, wv)[0]).all()
            assert not got[:r0 - at].any() and not got[r0 - at + 200:].any()
    m.free()
    buf.close()


def test_capture_refuses_to_make_a_matrix(dev, buf):
    """Its filling would be recorded, a memset among it. Refused before anything is queued: the
    capture goes on, its replays run what else it holds, and the same calls work after it."""
    from pagoda_amd import Matrix, PagodaError

    rng = np.random.default_rng(3)
    w = weights(rng, 48, 96)
    m, wv = matrix(dev, w), mx.values(*w)
    x = rng.normal(0, 1, (4, 96)).astype(np.float32)
    px, py, pc, ps = buf.up(x), buf.up(np.zeros((4, 48), np.float32)), buf.up(w[0]), buf.up(mx.padded(w[1], 16, np.uint8(0)))
    made = []

    def calls():
        for make in (lambda: Matrix.from_mxfp4_dev(dev, pc, 48, ps, 16, 48, 96), lambda: matrix(dev, w)):
            with pytest.raises(PagodaError) as e:
                made.append(make())
            assert e.value.code == -5
        m.gemv_dev(px, 96, 4, py, 48, F32)

    g = Graph(dev, calls)
    assert not made
    want, bound = x.astype(np.float64) @ wv.T, mx.product_bound(x.astype(np.float64), wv)
    for _ in range(3):
        put(dev, py, np.zeros((4, 48), np.float32))
        g.replay()
        assert (np.abs(buf.down(py, np.zeros((4, 48), np.float32)) - want) <= bound).all()
        for again in (Matrix.from_mxfp4_dev(dev, pc, 48, ps, 16, 48, 96), matrix(dev, w)):
            assert np.array_equal(again.dequant(), wv.astype(np.float32))
    g.close()
