"""8-bit KV attention to the accuracy of its terms (kv8_close.py), and over the range of f32: the smallest and
largest values, scores, queries and gates."""
import numpy as np
import pytest

import kv8
import kv8_close
from kv8 import BF16, F16, F32, PAGE, Step, typed, value
from kv8_close import assert_close
from test_gpu_kv8 import HEADS, Call, GpuPool, pool_of, queries
from test_gpu_mxfp4 import Buffers, buf  # noqa: F401

pytestmark = pytest.mark.gpu

# one chunk; several of them; verify rows; prompt rows; (last: attention over lists of all pages)
FORMS = {"decode": ([37, 250], [1, 1]), "chunks": ([3000, 90], [1, 1]), "verify": ([400, 30], [4, 3]),
         "prompt": ([150, 900], [70, 130]), "list": ([37, 800], [1, 2])}


def with_rows(step, k=None, v=None):
    """The step with other keys or values, f32 rows [positions, kv * hd] rounded to its type."""
    if k is not None:
        step.k_raw = typed(k, step.t)[0]
    if v is not None:
        step.v_raw = typed(v, step.t)[0]
    step.cache = kv8.Cache(step.cache.n, step.cache.kv, step.cache.hd)
    step.cache.append(value(step.k_raw, step.t), value(step.v_raw, step.t), step.slots)
    return step


def run(dev, buf, step, heads, t, q, gate=None, form="", pool=None):
    """Raw queries and gates of type t to results."""
    call = Call(dev, buf, step, pool or pool_of(dev, buf, step), heads, t, q, gate)
    if form != "list":
        return call.attn()
    return call.sparse(*call.select(step.width, 0, 0))


def some_rows(step, rng, most=40):
    rows = range(step.rows)
    return set(rows) if step.rows <= most else set(rng.choice(step.rows, most, replace=False)) | {0, step.rows - 1}


def check(dev, buf, rng, step, heads, t, q, qv, form="", gate=(None, None)):
    rows = some_rows(step, rng)
    want, off = kv8_close.attention(step, qv, heads, gate[1], rows=rows)
    assert np.isfinite(want[sorted(rows)]).all()
    got = run(dev, buf, step, heads, t, q, gate[0], form)
    rows = sorted(rows)
    assert_close(got[rows], want[rows], off[rows], t)
    return got, want


# ---- accuracy -----------------------------------------------------------------------------


@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [BF16, F16, F32])
def test_results_are_the_definitions_rounded(dev, buf, t, form, heads, kv, hd):
    """No result is another number of its type than one within the roundings of f32 sums and two f16 terms."""
    rng = np.random.default_rng(heads + hd + t + len(form))
    ctx, new = FORMS[form]
    step = Step(rng, kv, hd, ctx, new, t)
    q, qv, gate = queries(rng, step, heads, t, hd == 128)
    check(dev, buf, rng, step, heads, t, q, qv, form, gate)


# ---- the ends of the range -------------------------------------------------------------------


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("power", [-110, -118, -125])
def test_the_smallest_values(dev, buf, t, form, power):
    """Values whose pages have the lowest exponents come out as themselves."""
    rng = np.random.default_rng(-power)
    ctx, new = FORMS[form]
    step = Step(rng, 2, 64, ctx, new, t)
    with_rows(step, v=(rng.normal(0, 1, (len(step.slots), 128)) * 2.0 ** power).astype(np.float32))
    q, qv, _ = queries(rng, step, 6, t)
    got, want = check(dev, buf, rng, step, 6, t, q, qv, form)
    assert np.abs(got).max() > 2.0 ** (power - 3)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [F32, BF16])
def test_scores_of_large_queries_and_keys(dev, buf, t, form):
    """Queries of 2^100 beside keys of 2^60 that they have no channel in common with, and beside keys of 2^-100 that
    they do: all scores are small."""
    rng = np.random.default_rng(12)
    ctx, new = FORMS[form]
    heads, kv, hd = 6, 2, 64
    step = Step(rng, kv, hd, ctx, new, t)
    k = np.zeros((len(step.slots), kv, hd), np.float32)
    low = np.arange(len(k)) // PAGE % 2 == 0
    k[low, :, 0] = rng.normal(0, 1, (low.sum(), kv)) * 2.0 ** -98
    k[~low, :, 1:] = rng.normal(0, 1, ((~low).sum(), kv, hd - 1)) * 2.0 ** 60
    with_rows(step, k=k.reshape(len(k), -1))
    q = np.zeros((step.rows, heads, hd), np.float32)
    q[..., 0] = rng.normal(0, 1, (step.rows, heads)) * 2.0 ** 100
    q, qv = typed(q.reshape(step.rows, -1), t)
    check(dev, buf, rng, step, heads, t, q, qv.reshape(-1, heads, hd), form)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [16, 23, 26, 30, 60])
def test_scores_past_whole_numbers(dev, buf, t, form, power, sign):
    """Scores of about 2^power, all of one sign: nothing but the largest one's value is taken, whatever the spacing of
    f32 numbers there, from pages of different exponents."""
    rng = np.random.default_rng(power)
    ctx, new = FORMS[form]
    heads, kv, hd = 6, 2, 64
    step = Step(rng, kv, hd, ctx, new, t)
    n = len(step.slots)
    size = 2.0 ** rng.integers(-30, 30, n).repeat(PAGE)[:n, None]
    k = np.exp(rng.normal(0, 1, (n, 1)) + rng.normal(0, 0.1, (n, kv * hd)))
    with_rows(step, k=k.astype(np.float32), v=(rng.normal(0, 1, (n, kv * hd)) * size).astype(np.float32))
    q, qv = typed(np.abs(rng.normal(0, 1, (step.rows, heads * hd))) * sign * 2.0 ** (power - 3), t)
    check(dev, buf, rng, step, heads, t, q, qv.reshape(-1, heads, hd), form)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("power", [0, 16, 24, 27, 31])
def test_equal_scores_past_whole_numbers(dev, buf, form, power):
    """Positions of one key, whatever its score: the mean of their values, which lie in pages of very different
    exponents."""
    rng = np.random.default_rng(power + 1)
    ctx, new = FORMS[form]
    heads, kv, hd = 4, 1, 64
    step = Step(rng, kv, hd, ctx, new, F32)
    n = len(step.slots)
    key = np.abs(rng.normal(0, 1, (1, hd))) * 2.0 ** (power / 2)
    size = 2.0 ** rng.integers(-60, 60, n).repeat(PAGE)[:n, None]
    with_rows(step, k=np.repeat(key, n, 0).astype(np.float32), v=(rng.uniform(1, 2, (n, hd)) * size).astype(np.float32))
    for sign in (1, -1):
        q = (np.abs(rng.normal(0, 1, (step.rows, heads * hd))) * sign * 2.0 ** (power / 2)).astype(np.float32)
        got = run(dev, buf, step, heads, F32, q, form=form)
        v = step.cache.values(1)
        for row, s, seen in step.each_row():
            want = v[step.tables[s, :kv8.pages(seen)], 0].reshape(-1, hd)[:seen].mean(0)
            # (all values are positive: sums of n of them, and terms of the weights)
            assert (np.abs(got[row] - want) <= want * ((2 * seen + 16) * 2.0 ** -23 + 2.0 ** -20)).all()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("form", ["decode", "chunks", "prompt", "list"])
def test_infinite_queries_give_nan(dev, buf, t, form):
    """Also where all scores are the infinity that would be a masked position's."""
    rng = np.random.default_rng(14)
    ctx, new = FORMS[form]
    heads, kv, hd = 4, 2, 64
    step = Step(rng, kv, hd, ctx, new, t)
    k = np.abs(rng.normal(0, 1, (len(step.slots), kv * hd))) + 0.5
    with_rows(step, k=k.astype(np.float32))
    q, qv, _ = queries(rng, step, heads, t)
    q[0, 5], q[step.rows - 1, 3 * hd + 60] = [{BF16: np.uint16(b)}.get(t, x) for b, x in ((0xFF80, -np.inf), (0x7F80, np.inf))]
    got = run(dev, buf, step, heads, t, q, form=form)
    hit = np.zeros((step.rows, heads), bool)
    hit[0, 0] = hit[step.rows - 1, 3] = True
    assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("power", [-100, -118, -127, -135])
def test_the_smallest_queries(dev, buf, t, form, power):
    """Queries down to the smallest numbers before keys that are as large."""
    rng = np.random.default_rng(-power)
    ctx, new = FORMS[form]
    heads, kv, hd = 6, 2, 64
    step = Step(rng, kv, hd, ctx, new, t)
    size = 2.0 ** min(-power, 125)
    with_rows(step, k=(rng.normal(0, 1, (len(step.slots), kv * hd)).clip(-3, 3) * size).astype(np.float32))
    q, qv = typed(rng.normal(0, 1, (step.rows, heads * hd)) * 2.0 ** power, t)
    check(dev, buf, rng, step, heads, t, q, qv.reshape(-1, heads, hd), form)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [F32, BF16])
def test_gates_of_large_values(dev, buf, t, form):
    """A gate whose reciprocal lies below the normal range, before values that bring the product back."""
    rng = np.random.default_rng(15)
    ctx, new = FORMS[form]
    step = Step(rng, 2, 64, ctx, new, t)
    with_rows(step, v=(rng.normal(0, 1, (len(step.slots), 128)) * 2.0 ** 110).astype(np.float32))
    q, qv, _ = queries(rng, step, 6, t)
    g, gv = typed(rng.uniform(-88.5, -86.5, (step.rows, 6 * 64)), t)
    got, want = check(dev, buf, rng, step, 6, t, q, qv, form, (g, gv.reshape(-1, 6, 64)))
    assert np.abs(got).max() > 2.0 ** -20


def held(q, t):
    """Queries [rows, heads, hd] as the products take them: the head's largest entry brought to [2^14, 2^15) by a power of two,
    in two f16 terms (bf16 rows: one)."""
    e = np.frexp(np.abs(q).max(-1, keepdims=True))[1] - 15
    x = np.ldexp(q, -e)
    first = x.astype(np.float16).astype(float)
    return np.ldexp(first + ((x - first).astype(np.float16).astype(float) if t == F32 else 0), e)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [F32, BF16])
def test_scores_past_f32(dev, buf, t, form):
    """A head whose largest score is infinite is NaN, of either sign; infinitely low scores beside others count nothing."""
    rng = np.random.default_rng(16)
    ctx, new = FORMS[form]
    heads, kv, hd = 6, 2, 64
    step = Step(rng, kv, hd, ctx, new, t)
    n = len(step.slots)
    k = np.zeros((n, kv, hd), np.float32)
    k[..., 0] = rng.uniform(1, 2, (n, kv)) * 2.0 ** 60
    k[:, 1, 1:] = np.where(np.arange(n) % 3 == 0, 1, 0)[:, None] * rng.normal(0, 1, (n, hd - 1)) * 2.0 ** 55
    k[::3, 1, 0] = 0  # head 1: every third position has scores of its own
    with_rows(step, k=k.reshape(n, -1))
    q = np.zeros((step.rows, heads, hd), np.float32)
    q[:, :3, 0] = np.where(np.arange(3) == 1, 1, -1) * 2.0 ** 100
    q[:, 3:, 0] = -(2.0 ** 100)
    q[:, 3:, 1:] = rng.normal(0, 1, (step.rows, 3, hd - 1)) * 2.0 ** 67  # (far apart, and far below 2^127 more)
    q, qv = typed(q.reshape(step.rows, -1), t)
    qv = qv.reshape(-1, heads, hd)
    got = run(dev, buf, step, heads, t, q, form=form)
    assert np.isnan(got[:, :3]).all()
    rows = sorted(some_rows(step, rng))
    # Entries of 2^67 beside 2^100 are held to 2^61, half of f16's smallest step times 2^86: scores of 2^122 move by
    # 2^116 then, which may be more than the two largest lie apart.
    largest = np.abs(qv).max(-1, keepdims=True)
    assert (np.abs(held(qv, t) - qv) <= np.maximum(2.0 ** -22 * np.abs(qv), 2.0 ** -39 * largest)).all()
    want, off = kv8_close.attention(step, held(qv, t), heads, rows=rows)
    assert_close(got[rows, 3:], want[rows, 3:], off[rows, 3:], t)
