"""The 8-bit KV cache at more than 64 sequences (the lanes that look through them at once) with contexts that are cut, and the
choice among many different scores."""
import numpy as np
import pytest

import kv8
import kv8_close
from kv8 import BF16, F16, F32, PAGE, Step, typed, value
from kv8_close import assert_close
from test_gpu_kv8 import Call, GpuPool, pool_of, queries
from test_gpu_mxfp4 import Buffers, buf  # noqa: F401

pytestmark = pytest.mark.gpu


def sequences(rng, n, most):
    """Contexts of 1 to 600 positions, the longest on both sides of every 64th sequence, with up to `most` rows and
    some with none."""
    ctx = np.exp(rng.uniform(0, np.log(600), n)).astype(int) + 1
    ctx[[0, 61, 62, 63, n - 2, n - 1]] = [500, 3, 1, 900, 700, 650]
    new = np.where(rng.random(n) < 0.15, 0, np.where(rng.random(n) < 0.9, 1, rng.integers(1, most + 1, n)))
    new[[63, n - 2, n - 1]] = [most, most, most]
    return ctx.tolist(), np.minimum(new, ctx).tolist()


@pytest.mark.parametrize("n", [65, 150, 257])
@pytest.mark.parametrize("t,heads,kv,hd,most", [(F32, 6, 1, 64, 1), (BF16, 7, 1, 128, 4), (F16, 12, 2, 64, 15), (F32, 7, 1, 64, 60)])
def test_cut_contexts_of_many_sequences(dev, buf, n, t, heads, kv, hd, most):
    """Decode rows, verify rows, and rows of both kernels in one call."""
    rng = np.random.default_rng(n + most)
    ctx, new = sequences(rng, n, most)
    step = Step(rng, kv, hd, ctx, new, t)
    q, qv, (g, gv) = queries(rng, step, heads, t, True)
    want, off = kv8_close.attention(step, qv, heads, gv)
    call = Call(dev, buf, step, pool_of(dev, buf, step), heads, t, q, g)
    got = call.attn()
    assert_close(got, want, off, t)
    assert np.array_equal(call.attn(), got)


@pytest.mark.parametrize("n", [65, 150])
@pytest.mark.parametrize("t,heads,kv,hd", [(F32, 6, 2, 64), (F16, 4, 1, 128)])
def test_selection_of_many_sequences(dev, buf, n, t, heads, kv, hd):
    rng = np.random.default_rng(n + hd)
    ctx, new = sequences(rng, n, 3)
    step = Step(rng, kv, hd, ctx, new, t)
    q, qv, _ = queries(rng, step, heads, t)
    call = Call(dev, buf, step, pool_of(dev, buf, step), heads, t, q)
    for top in (5, 24):
        picked = kv8.select(step, qv, heads, top, 1, 2 if top > 5 else 0)
        sel, count = call.select(top, 1, 2 if top > 5 else 0)
        for row in range(step.rows):
            for h in range(kv):
                assert sel[row, h].tolist() == picked[row][h] + [-1] * (top - len(picked[row][h])), (row, h)
                assert count[row, h] == len(picked[row][h])
        want, off = kv8_close.attention(step, qv, heads, None, picked)
        assert_close(call.sparse(sel, count), want, off, t)


def chosen(score, top, sinks, recent):
    pages = np.arange(len(score))
    forced = (pages < sinks) | (pages >= len(score) - recent)
    return np.sort(np.lexsort((pages, -score, ~forced))[:top])


@pytest.mark.parametrize("kind", ["spread", "crowded", "steps"])
@pytest.mark.parametrize("pages", [5000, 9100])
def test_selection_among_different_scores(dev, buf, kind, pages):
    """Thousands of different scores, fewer and more than threads hold: spread over the bins that a round counts; nearly all
    in one bin beside a few far out, so that its keys need a round of their own; and in steps of very different size."""
    rng = np.random.default_rng(pages)
    key = np.zeros((pages, 64))
    channels = rng.integers(0, 450, (pages, 64))
    if kind == "spread":
        key[:] = channels
    elif kind == "crowded":
        # (the outliers make the range of scores' bits so wide that the others share a bin or two)
        key[:] = 448
        key[:, 48:] = 256 + 32 * (channels[:, 48:] % 7)
        key[rng.choice(pages, 9, replace=False)] *= 2.0 ** 60
        key[rng.choice(pages, 9, replace=False)] *= -1
    else:
        key[:] = channels * 2.0 ** rng.integers(-100, 100, (pages, 1))
    k = key.repeat(PAGE, 0).astype(np.float32)
    k[:, -1] = np.where(k[:, -1] == 0, k[:, 0], k[:, -1])
    slots = np.arange(PAGE * pages, dtype=np.int32)
    pool = GpuPool(dev, buf, 1, 64, pages)
    pool.append(k, k, slots, F32)
    q = np.abs(rng.normal(0, 1, (1, 64))).astype(np.float32)
    # the definition, page by page at once: an exponent, codes, bounds in steps of 4, a sum of whole numbers
    first = k[::PAGE].astype(float)
    exps = np.array([kv8.holds(x) for x in np.abs(first).max(1)], float)
    codes = kv8.round_e4m3(first * 2.0 ** -exps[:, None]) / 4
    q8 = np.rint(q[0].astype(float) * 2.0 ** -kv8.holds(np.abs(q).max(), 127.0))
    score = np.maximum(q8 * np.ceil(codes), q8 * np.floor(codes)).sum(1) * 2.0 ** exps
    assert len(np.unique(score)) > 1024
    table = rng.permutation(pages).astype(np.int32)
    ptrs = [buf.up(a) for a in (q, np.int32([0, 1]), np.int32([pages * PAGE]), table)]
    for top, sinks, recent in ((1, 0, 0), (40, 1, 2), (700, 0, 0), (2500, 5, 3), (pages - 1, 0, 1)):
        sel, count = np.full(top, 9, np.int32), np.int32([9])
        ps, pc = buf.up(sel), buf.up(count)
        size = pool.pool.sparse_ws_bytes(1, 1, pages, top)
        pool.pool.select_dev(1, ptrs[0], 64, F32, 1, *ptrs[1:], pages, 1, top, sinks, recent, ps, pc,
                             buf.up(np.zeros(size, np.uint8)), size)
        assert buf.down(pc, count)[0] == top
        np.testing.assert_array_equal(buf.down(ps, sel), chosen(score[table], top, sinks, recent), err_msg=str(top))


def test_a_workspace_of_the_largest_step_serves_smaller_ones(dev, buf):
    rng = np.random.default_rng(70)
    heads, kv, hd, top = 24, 4, 64, 128
    width = 140
    for rows in (1, 20, 96):
        step = Step(rng, kv, hd, [width * PAGE] if rows < 20 else [2100, 40], [rows] if rows < 20 else [1, rows - 1], F16)
        q, qv, _ = queries(rng, step, heads, F16)
        pool = pool_of(dev, buf, step)
        call = Call(dev, buf, step, pool, heads, F16, q)
        size = max(pool.pool.sparse_ws_bytes(heads, 256, width + 9, t) for t in (top, top + 9))
        call.workspace = lambda t: (buf.up(np.full(size, 0xFF, np.uint8)), size)
        picked = kv8.select(step, qv, heads, top, 0, 1)
        sel, count = call.select(top, 0, 1)
        assert all(sel[r, h, :count[r, h]].tolist() == picked[r][h] for r in range(rows) for h in range(kv))
        want, off = kv8_close.attention(step, qv, heads, None, picked)
        assert_close(call.sparse(sel, count), want, off, F16)


@pytest.mark.parametrize("t,heads,kv,hd", [(F32, 24, 4, 256), (BF16, 28, 4, 128), (F16, 14, 2, 64)])
@pytest.mark.parametrize("ctx,new", [([6000, 300], [1, 1]), ([3000, 40], [4, 2]), ([2500, 300], [40, 1]), ([9000], [1])])
def test_attention_stays_in_its_workspace(dev, buf, t, heads, kv, hd, ctx, new):
    """Of the size that the call's largest number of rows needs, with the bytes behind it left as they were."""
    rng = np.random.default_rng(ctx[0] + hd)
    step = Step(rng, kv, hd, ctx, new, t)
    q, qv, _ = queries(rng, step, heads, t)
    call = Call(dev, buf, step, pool_of(dev, buf, step), heads, t, q)
    p = call.pool.pool
    rows = sorted({0, step.rows - 1} | set(rng.choice(step.rows, min(step.rows, 9), replace=False)))
    want, off = kv8_close.attention(step, qv, heads, rows=rows)
    for most in (max(new), 1):
        size = p.attn_ws_bytes(heads, len(ctx), step.width, step.rows, most)
        assert size <= p.attn_ws_bytes(heads, len(ctx), step.width, step.rows)
        whole = np.full(size + 65536, 0xFF, np.uint8)
        ws = buf.up(whole)
        p.attn_dev(*call.args(), most, call.out, call.fresh.shape[1], ws, size)
        assert_close(call.result()[rows], want[rows], off[rows], t)
        assert (buf.down(ws, whole)[size:] == 0xFF).all()


@pytest.mark.parametrize("t,heads,kv,hd", [(F32, 6, 2, 64), (BF16, 20, 1, 128), (F16, 3, 3, 256)])
def test_listed_pages_behind_a_rows_context(dev, buf, t, heads, kv, hd):
    """Entries of the table past a row's context, which may name pages that hold anything, or nothing yet: a list that names
    them gives what it gives without them."""
    rng = np.random.default_rng(hd)
    step = Step(rng, kv, hd, [300, 70, 40], [4, 1, 1], t, spare=9, widen=8)
    pool = pool_of(dev, buf, step)  # (pages not written hold 0xFF, codes of no number)
    used = set(step.slots // PAGE)
    fresh = [p for p in range(step.cache.n) if p not in used]
    for s, c in enumerate(step.ctx):
        m = kv8.pages(c)
        step.tables[s, m:] = rng.choice(fresh + [-1, step.cache.n], step.width - m)
        step.tables[s, m:m + 4] = fresh[:4]
    q, qv, _ = queries(rng, step, heads, t)
    call = Call(dev, buf, step, pool, heads, t, q)
    for top in (7, 60):
        sel = rng.integers(0, step.width, (step.rows, kv, top)).astype(np.int32)
        sel[..., -1] = step.width - 1
        sel[..., 0] = 0
        picked = {r: [[p for p in sel[r, h] if p * PAGE < seen] for h in range(kv)] for r, _, seen in step.each_row()}
        got = call.sparse(sel, np.full((step.rows, kv), top, np.int32))
        want, off = kv8_close.attention(step, qv, heads, None, picked)
        assert_close(got, want, off, t)


def test_the_f32_attention_refuses_rows_to_spare(dev, buf):
    """Rows that a step's maps give to no sequence are an error there, before anything is read for them."""
    import ctypes as C

    from pagoda_amd import PagodaError
    from pagoda_amd._lib import call
    from pagoda_amd.kv8 import kv_tables_dev

    ints = lambda *v: buf.up(np.int32(v))
    tables, rows = buf.up(np.full((1, 4), -1, np.int32)), 5
    outs = [buf.up(np.zeros(n, np.int32)) for n in (1, 1, 2, rows, rows, rows, 1)]
    kv_tables_dev(dev, 16, 1, ints(0), ints(3), tables, 4, ints(1, 0), 2, ints(0), rows, *outs)
    assert buf.down(outs[3], np.zeros(rows, np.int32)).tolist() == [0, 0, 0, -1, -1]
    q = np.ones((rows, 2, 64), np.float32)
    pool, out = buf.up(np.ones((2, 1, 16, 64), np.float32)), buf.up(q)
    attend = lambda n: call("pgd_attn_decode_dev", dev.handle, 2, 1, 64, 16, C.c_void_p(buf.up(q)), None, C.c_void_p(pool),
                            C.c_void_p(pool), C.c_void_p(outs[3]), C.c_void_p(outs[4]), C.c_void_p(tables), 4, n, C.c_void_p(out))
    with pytest.raises(PagodaError):
        attend(rows)
    attend(3)
    assert np.allclose(buf.down(out, q)[:3], 1)


@pytest.mark.parametrize("t,heads,kv,hd", [(F32, 6, 2, 64), (BF16, 7, 1, 128), (F16, 12, 2, 256)])
def test_results_do_not_hang_on_pages_of_others(dev, buf, t, heads, kv, hd):
    """The pool's first page, which no sequence here has, changes no bit of a result, whatever it holds: contexts and
    lists of odd numbers of pages among them."""
    rng = np.random.default_rng(80 + hd)
    for ctx, new in (([37, 300, 1], [1, 1, 1]), ([90, 3000], [4, 1]), ([700, 75], [150, 11])):
        step = Step(rng, kv, hd, ctx, new, t)
        q, qv, _ = queries(rng, step, heads, t)
        pool = GpuPool(dev, buf, kv, hd, step.cache.n + 1)
        pool.append(step.k_raw, step.v_raw, step.slots + PAGE, t)
        step.tables = np.where(step.tables >= 0, step.tables + 1, -7).astype(np.int32)
        call = Call(dev, buf, step, pool, heads, t, q)
        sel = np.stack([rng.permutation(step.width)[:3] for _ in range(step.rows * kv)]).reshape(step.rows, kv, 3).astype(np.int32)
        sel[..., 0] = 0
        count = np.full((step.rows, kv), 3, np.int32)
        first = None
        for size in (None, 0.0, 1.0, 2.0 ** 15, 2.0 ** -14):  # (as it was allocated, then written)
            if size is not None:
                rows = typed(np.full((PAGE, kv * hd), size) * rng.choice([-1, 1], (PAGE, kv * hd)), t)[0]
                pool.append(rows, rows, np.arange(PAGE), t)
            if size == 2.0 ** 15 and t != F16:
                rows = typed(rows.astype(np.float32) if t == F32 else value(rows, t) * 2.0 ** 100, t)[0]
                pool.append(rows, rows, np.arange(PAGE), t)
            got = call.attn(), call.sparse(sel, count)
            first = first or got
            for a, b in zip(got, first):
                assert np.array_equal(a, b), (ctx, size)
