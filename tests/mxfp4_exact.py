"""Rows and MXFP4 weights whose products are exact in f32 whatever the order of the sums,
so that outputs are compared bit for bit and a lost term, digit or k tile shows.

Products of whole numbers x (f32 rows: of 2^s times whole numbers) with weights in halves:
every partial sum, and that of any leading terms or digits of x (at most twice x each), is a
whole number of halves below 2^24. Each row and each output has a power of two of its own."""
import numpy as np

import mxfp4 as mx
from mxfp4_choice import BF16, F16, F32, PLANES

BUDGET = 1 << 22  # halves, of a sum of magnitudes
OUTLIER = 2.0 ** 28  # steps of a row's digits are 1 beside it: 2^(28 - 28)


def _scales(rng, n, k, e):
    """Scale bytes 2^e[row] times 1 or 2."""
    return (127 + e[:, None] + rng.integers(0, 2, (n, k // 32))).astype(np.uint8)


def dense_weights(rng, n, k):
    """Codes of every value; each block's first element zero."""
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    codes[:, 0::16] &= 0xF0
    return codes, _scales(rng, n, k, rng.integers(-3, 4, n))


def dense_rows(rng, t, rows, k, e):
    """Rows 2^e[row] times whole numbers of every column. f32: three rows of four have an
    outlier under each block's zero weight, and small numbers in digits 4 and 5, 3 and 4, or 2
    and 3; the others (and other types) have the numbers alone. What the call takes, values."""
    if t == PLANES:
        p = rng.integers(0, 256, (rows, k // 2), dtype=np.uint8), _scales(rng, rows, k, e)
        return p, mx.values(*p)
    top = min(BUDGET // (24 * k), 255 if t == BF16 else 2047)
    x = rng.integers(-top, top + 1, (rows, k)).astype(np.float64)
    if t == F32:
        kind = np.arange(rows) % 4
        x *= 2.0 ** np.array([0, 0, 8, 16])[kind][:, None]
        x[:, 0::32] = np.where(kind[:, None] > 0, OUTLIER, x[:, 0::32])
    raw, v = mx.rows_of((x * 2.0 ** e[:, None]).astype(np.float32), t)
    assert np.array_equal(v, x * 2.0 ** e[:, None])
    return raw, x * 2.0 ** e[:, None]


def sparse_weights(rng, n, k):
    """Powers of two of either sign and zeros; each block's first element zero."""
    code = np.array([0, 1, 2, 4, 6, 9, 10, 12, 14, 1, 2, 4, 6, 9, 10, 12], np.uint8)
    c = code[rng.integers(0, 16, (n, k))]
    c[:, 0::32] = 0
    return c[:, 0::2] | (c[:, 1::2] << 4), _scales(rng, n, k, rng.integers(-3, 4, n))


def sparse_rows(rng, t, rows, k, e):
    """One number of all its type's bits a row, the lowest set; f32: odd rows have 20 bits of
    it beside an outlier (digits 1 to 5), the others 24 (digits 0 to 4)."""
    bits = {F32: 24, F16: 11, BF16: 8}[t]
    r, col = np.arange(rows), rng.integers(0, k // 32, rows) * 32 + rng.integers(1, 32, rows)
    v = (rng.integers(1 << (bits - 1), 1 << bits, rows) | 1).astype(np.int64)
    x = np.zeros((rows, k))
    if t == F32:
        v |= 0x4181  # (each of three terms)
        odd = r % 2 == 1
        v = np.where(odd, v & 0xFFFFF, v)
        x[r, col // 32 * 32] = np.where(odd, OUTLIER, 0)
    x[r, col] = v * np.where(rng.random(rows) < 0.5, -1, 1)
    raw, f = mx.rows_of((x * 2.0 ** e[:, None]).astype(np.float32), t)
    assert np.array_equal(f, x * 2.0 ** e[:, None])
    return raw, x * 2.0 ** e[:, None]


def exponents(rng, t, rows, pair=False):
    """Rows' powers of two: small ones for a pair, so that most gates are where silu is neither 0
    nor its argument; f16 rows in their normal range."""
    if pair:
        return rng.integers(-40, -17, rows)
    return rng.integers(-3, 4, rows) if t == F16 else rng.integers(-20, 21, rows)


def terms(x, count):
    """bf16 terms of f32 values, each the truncation of what is left."""
    out, rest = [], np.asarray(x, np.float32)
    for _ in range(count):
        h = (rest.view(np.uint32) & 0xFFFF0000).view(np.float32)
        out.append(h.astype(np.float64))
        rest = rest - h
    return out


def digits(x):
    """Six base-32 digits of f32 rows as values, by block of 32: whole numbers of steps 2^(e -
    28), 2^e the largest magnitude's power of two, digits -15 to 16 (the top one -16 to 16)."""
    b = np.asarray(x, np.float64).reshape(x.shape[0], -1, 32)
    top = np.abs(b).max(-1, keepdims=True)
    step = 2.0 ** (np.floor(np.log2(np.where(top > 0, top, 1))) - 28)
    n = np.rint(b / step).astype(np.int64)
    out = []
    for i in range(5):
        d = (n + 15) % 32 - 15
        out.append(d * 32.0 ** i * step)
        n = (n - d) // 32
    out.append(n * 32.0 ** 5 * step)
    return [d.reshape(x.shape) for d in out[::-1]]
