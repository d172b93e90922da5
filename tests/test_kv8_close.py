"""The bound that attention over the 8-bit cache is held to (kv8_close.py), on the CPU: plain f32 arithmetic and rows in
two f16 terms keep it, and rows or weights in one f16 term do not."""
import numpy as np
import pytest

import kv8_close
from kv8 import BF16, F16, F32, PAGE, Step, pages, typed, value


def held(x, bits):
    """To so many bits, to nearest."""
    m, e = np.frexp(x)
    return np.ldexp(np.rint(np.ldexp(m, bits)), e - bits)


def computed(step, q, heads, q_bits, weight_bits):
    """In f32, with queries and weights held to so many bits."""
    c = step.cache
    g = heads // c.kv
    out = np.zeros((step.rows, heads, c.hd), np.float32)
    for row, s, seen in step.each_row():
        for h in range(heads):
            k, v = (c.values(w)[step.tables[s, :pages(seen)], h // g].reshape(-1, c.hd)[:seen].astype(np.float32) for w in range(2))
            if seen:
                x = k @ held(q[row, h], q_bits).astype(np.float32) * np.float32(1 / np.sqrt(c.hd))
                w = np.exp(x - x.max())
                out[row, h] = held(w, weight_bits).astype(np.float32) @ v / w.sum(dtype=np.float32)
    return out


SHAPES = [(F32, 6, 2, 64, [40, 300, 1], [3, 1, 1], 1.0), (F32, 6, 1, 256, [33, 5003], [2, 1], 1.0), (F16, 8, 4, 128, [700], [1], 1.0),
          (BF16, 6, 1, 256, [900, 17], [2, 1], 1.0), (F32, 4, 2, 128, [70, 300], [2, 1], 30.0), (BF16, 4, 2, 128, [300], [2], 1e-3)]


@pytest.mark.parametrize("t,heads,kv,hd,ctx,new,scale", SHAPES)
def test_what_the_bound_takes_and_rejects(t, heads, kv, hd, ctx, new, scale):
    rng = np.random.default_rng(hd + ctx[0])
    step = Step(rng, kv, hd, ctx, new, t)
    q = typed(rng.normal(0, scale, (step.rows, heads * hd)), t)[1].reshape(-1, heads, hd)
    want, off = kv8_close.attention(step, q, heads)

    def ok(q_bits, weight_bits):
        got = value(typed(computed(step, q, heads, q_bits, weight_bits), t)[0], t)
        return kv8_close.within(got, want, off, t)

    assert ok(24, 24).all() and ok(22, 21).all()
    if scale <= 1:  # (past that the scores' own roundings in f32 are larger than those of weights)
        assert not ok(24, 11).all()
    if t == F32:
        # at flat and at steep softmaxes, for a good part of the results
        assert (~ok(11, 24)).mean() > 0.1


def test_one_position_takes_all():
    """At scores far apart nothing but the largest one's value is taken."""
    rng = np.random.default_rng(3)
    step = Step(rng, 2, 128, [70, 300], [2, 1], F32)
    q = typed(rng.normal(0, 1e4, (3, 4 * 128)), F32)[1].reshape(3, 4, 128)
    want, off = kv8_close.attention(step, q, 4)
    assert (off <= 1e-4 * np.abs(want).max(-1, keepdims=True)).mean() > 0.9
    for wrong in (np.zeros_like(want), np.full_like(want, 1e6), want * 1.001):
        assert not kv8_close.within(wrong.astype(np.float32), want, off, F32).any(-1).all()
    assert kv8_close.within(computed(step, q, 4, 24, 24), want, off, F32).all()
