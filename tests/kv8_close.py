"""How near attention over the 8-bit cache has to be to its definition: what each position's
score and weight may be off by itself, not the worst position's for all.

A score is a sum of 2 hd products in f32 (f32 rows enter as two terms). An addition is off by up to 2^-24 of the
sum so far, and sums of products of no common sign stay of the size of `spread`, the root of the sum of their squares: 2^-24
sqrt(2 hd) spread in the root mean square at most. q is held to 2^-22 of each entry: 2^-22 spread. The product with the scale
and the difference from the largest score are rounded to f32: 2^-23 of the score. A weight: 2^-21 (its two terms) and
2^-22 (exp2), together less than 2^-20. All of these are independent from position to position, so a result, whose derivative by score j is
w_j (v_j - o), is off by the root of the sum of squares; SURE times that is allowed. The sums over n positions and the
joining of parts: (sqrt(n) + 16) 2^-23 of the result and of the spread of what is summed, four times."""
import numpy as np

import kv8
from kv8 import PAGE, pages, typed, value

SURE = 6


def attend(q, k, v, unit):
    """One query [hd] over positions k, v [n, hd] (float64), unit the power of two of each position's value
    codes: the result, and how far it may be off before it is rounded to its type."""
    n, hd = k.shape
    if n == 0:
        return np.zeros(hd), np.zeros(hd)
    prod = k * q / np.sqrt(hd)
    s = prod.sum(1)
    d = (2.0 ** -24 * np.sqrt(2 * hd) + 2.0 ** -22) * np.sqrt((prod ** 2).sum(1)) + 2.0 ** -23 * np.abs(s) + 2.0 ** -20
    w = np.exp(s - s.max())
    w /= w.sum()
    o = w @ v
    d = np.minimum(SURE * d, 40)
    off = np.sqrt(((w * np.expm1(d)) ** 2) @ (v - o) ** 2) / (w @ np.exp(-d))
    spread = np.sqrt(w ** 2 @ v ** 2)
    # f16 terms hold nothing below 2^-36 of the largest weight of a code; codes are up to 448
    least = SURE * np.sqrt(n) * 448 * 2.0 ** -36 * (w * unit).max()
    return o, off + 4 * (np.sqrt(n) + 16) * 2.0 ** -23 * (np.abs(o) + spread) + least


def attention(step, q, heads, gate=None, picked=None, rows=None):
    """float64 results [rows, heads, hd] and how far they may be off before they are rounded; picked: (row, kv head) ->
    places in the table; rows: those that are wanted (the others NaN)."""
    c = step.cache
    g = heads // c.kv
    out, off = (np.full((step.rows, heads, c.hd), np.nan) for _ in range(2))
    kv = [c.values(w) for w in range(2)]
    for row, s, seen in step.each_row():
        if rows is not None and row not in rows:
            continue
        for h in range(heads):
            head = h // g
            places = np.arange(pages(seen)) if picked is None else np.asarray(picked[row][head], int)
            at = (places[:, None] * PAGE + np.arange(PAGE)).reshape(-1)
            use = at < seen
            kk, vv = (x[step.tables[s, places], head].reshape(-1, c.hd)[use] for x in kv)
            unit = 2.0 ** c.exps[1, step.tables[s, places], head].astype(float).repeat(PAGE)[use]
            o, b = attend(q[row, h], kk, vv, unit)
            if gate is not None:
                sg = kv8.sigmoid(gate[row, h])
                # exp2 of a rounded product, a sum, a quotient
                b = b * sg + np.abs(o) * sg * (8 + 2 * np.abs(gate[row, h])) * 2.0 ** -24
                o = o * sg
            out[row, h], off[row, h] = o, b
    return out, off


def within(got, want, off, t):
    """Whether results are what some value within `off` of the wanted one rounds to (a f32 sum is held to 2^-149 too)."""
    off = off + 2.0 ** -149
    ends = []
    with np.errstate(over="ignore"):
        for x in (want - off, want + off):
            # (to f32 first, as the sums are)
            ends.append(value(typed(x, t)[0], t))
    return (ends[0] <= got) & (got <= ends[1])


def assert_close(got, want, off, t):
    bad = ~within(got, want, off, t)
    assert not bad.any(), (bad.mean(), np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], off[bad][:5])
