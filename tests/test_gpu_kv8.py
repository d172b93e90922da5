"""The 8-bit paged KV cache on the GPU against its definition (kv8.py): codes, tables and selections
exactly, attention within the bound of its f32 sums."""
import numpy as np
import pytest

import kv8
from kv8 import BF16, F16, F32, PAGE, Step, typed, value
from test_gpu_mxfp4 import Buffers, buf  # noqa: F401

pytestmark = pytest.mark.gpu

HEADS = [(14, 2, 64), (4, 4, 64), (28, 4, 128), (24, 4, 256), (40, 2, 128), (3, 3, 256)]


def strided(a, ld, fill):
    """Rows at a stride of ld elements, fill between them."""
    out = np.full((a.shape[0], ld), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


class GpuPool:
    """A pool whose memory holds 0xFF everywhere before its first use."""

    def __init__(self, dev, buf, kv, hd, n_pages):
        from pagoda_amd import Kv8Pool
        from pagoda_amd.kv8 import page_bytes

        self.raw = np.full(n_pages * page_bytes(kv, hd) + 64, 0xFF, np.uint8)
        self.at = buf.up(self.raw)
        self.dev, self.buf, self.kv, self.hd = dev, buf, kv, hd
        self.pool = Kv8Pool(dev, kv, hd, n_pages, self.at)

    def append(self, k, v, slots, t, ldk=0, ldv=0):
        """Raw rows of type t."""
        ldk, ldv = ldk or k.shape[1], ldv or v.shape[1]
        self.pool.append_dev(self.buf.up(strided(k, ldk, k.dtype.type(7))), ldk,
                             self.buf.up(strided(v, ldv, v.dtype.type(7))), ldv, t, self.buf.up(np.int32(slots)), len(slots))

    def read(self, slots, ld=0, fill=-77.0):
        width = self.kv * self.hd
        ld = ld or width
        k, v = (np.full((len(slots), ld), fill, np.float32) for _ in range(2))
        pk, pv = self.buf.up(k), self.buf.up(v)
        self.pool.read_dev(self.buf.up(np.int32(slots)), len(slots), pk, ld, pv, ld)
        k, v = self.buf.down(pk, k), self.buf.down(pv, v)
        assert (k[:, width:] == fill).all() and (v[:, width:] == fill).all()
        return k[:, :width], v[:, :width]

    def untouched(self):
        return np.array_equal(self.buf.down(self.at, self.raw)[-64:], self.raw[-64:])


def pool_of(dev, buf, step):
    p = GpuPool(dev, buf, step.cache.kv, step.cache.hd, step.cache.n)
    if len(step.slots):
        p.append(step.k_raw, step.v_raw, step.slots, step.t)
    return p


def same_as(cache, pool, slots):
    for got, w in zip(pool.read(slots), range(2)):
        with np.errstate(over="ignore"):  # (the largest f32 rounds to a code times 2^120 past it)
            np.testing.assert_array_equal(got, cache.read(w, slots).astype(np.float32))


# ---- writing and reading ---------------------------------------------------------------


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("kv,hd", [(1, 64), (3, 64), (2, 128), (4, 256)])
def test_pages_fill_in_steps(dev, buf, t, kv, hd):
    """Prompts, single tokens and chunks of several sequences, padding rows among them, over magnitudes that make
    pages grow: after every call all that was written reads back bit for bit."""
    rng = np.random.default_rng(kv * hd + t)
    cache, pool = kv8.Cache(12, kv, hd), GpuPool(dev, buf, kv, hd, 12)
    tables = rng.permutation(12).reshape(3, 4)
    lens = [0, 0, 0]
    for counts in ((17, 1, 0), (1, 1, 15), (1, 30, 1), (13, 1, 3), (0, 5, 1), (31, 0, 44)):
        slots = []
        for s, n in enumerate(counts):
            p = np.arange(lens[s], lens[s] + n)
            slots += list(tables[s, p // PAGE] * PAGE + p % PAGE)
            lens[s] += n
            slots += [-1] * (s == 1)
        size = 2.0 ** rng.integers(-12, 6, (2, len(slots), 1)) * rng.normal(0, 1, (2, len(slots), kv * hd))
        (kr, k), (vr, v) = typed(size[0], t), typed(size[1], t)
        pool.append(kr, vr, slots, t, kv * hd + 8, kv * hd + 24)
        cache.append(k, v, slots)
        live = [tables[s, p // PAGE] * PAGE + p % PAGE for s in range(3) for p in range(lens[s])]
        same_as(cache, pool, live)
    assert pool.untouched()


def edge_rows(rng, width):
    """Rows of one binade's codes, ties and neighbours of ties, the smallest and largest numbers, zeros."""
    codes = np.array([m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)])[:127]
    mid = (codes[1:] + codes[:-1]) / 2
    pts = np.concatenate([codes, mid, mid * (1 + 2.0 ** -23), mid * (1 - 2.0 ** -23)])
    rows = []
    for scale in (1.0, 2.0 ** -30, 2.0 ** 100, 2.0 ** -126, 2.0 ** -140):
        for _ in range(3):
            x = rng.choice(pts, width) * rng.choice([-1, 1], width) * scale
            x[0] = 448 * scale
            rows.append(x)
    rows.append(np.zeros(width))
    rows.append(rng.choice([1e-45, -1e-45, 1e-38, 0.0, -0.0], width))
    rows.append(np.finfo(np.float32).max * np.linspace(-1, 1, width))
    rows.append(448 * 2.0 ** rng.integers(-149, 119, width).astype(np.float64) * rng.uniform(0.5, 1, width))
    return np.array(rows, np.float64).astype(np.float32)


@pytest.mark.parametrize("together", [False, True])
def test_codes_at_their_edges(dev, buf, together):
    """Every row a page of its own, and rows of all magnitudes in one page."""
    rng = np.random.default_rng(5 + together)
    x = edge_rows(rng, 256)
    if together:
        x = x[rng.permutation(len(x))[:16]]
        x = x[np.argsort(np.abs(x).max(1))]  # (the page grows with every row)
        slots = list(range(16, 32))
    else:
        slots = list(range(16, 16 * (len(x) + 1), 16))
    cache, pool = kv8.Cache(len(x) + 1, 2, 128), GpuPool(dev, buf, 2, 128, len(x) + 1)
    v = x[::-1].copy()
    if together:
        for i in range(16):
            pool.append(x[i:i + 1], v[i:i + 1], slots[i:i + 1], F32)
            cache.append(x[i:i + 1].astype(float), v[i:i + 1].astype(float), slots[i:i + 1])
    else:
        pool.append(x, v, slots, F32)
        cache.append(x.astype(float), v.astype(float), slots)
    same_as(cache, pool, slots)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_nonfinite_rows_stay_in_their_place(dev, buf, t):
    rng = np.random.default_rng(t)
    bad = {F32: [np.inf, -np.inf, np.nan], F16: [np.inf, -np.inf, np.nan], BF16: [0x7F80, 0xFF80, 0x7FC1]}[t]
    raw = [typed(rng.normal(0, 1, (14, 256)), t)[0].copy() for _ in range(2)]
    raw[0][2, 5], raw[1][6, 200], raw[0][13, 255] = bad  # heads 0, 3, 3 of 4
    raw[1][13, 0] = bad[0]
    cache, pool = kv8.Cache(2, 4, 64), GpuPool(dev, buf, 4, 64, 2)
    k, v = (value(x, t) for x in raw)
    for part in (slice(0, 7), slice(7, 9), slice(9, 14)):
        s = np.arange(16, 30)[part]
        pool.append(raw[0][part], raw[1][part], s, t)
        cache.append(k[part], v[part], s)
    same_as(cache, pool, np.arange(16, 30))
    assert np.isnan(pool.read([18])[1][0, :64]).all() and not np.isnan(pool.read([18])[1][0, 64:]).any()
    # written again from a place before them, the flags go
    good = typed(rng.normal(0, 1, (2, 256)), t)
    pool.append(good[0], good[0], [17, 18], t)
    cache.append(good[1], good[1], [17, 18])
    same_as(cache, pool, [16, 17, 18])


def test_slots_outside_the_pool(dev, buf):
    """Left out by the write, left as they were by the read."""
    rng = np.random.default_rng(1)
    x = rng.normal(0, 1, (6, 64)).astype(np.float32)
    cache, pool = kv8.Cache(2, 1, 64), GpuPool(dev, buf, 1, 64, 2)
    slots = [-1, 0, 32, 33, 16, 2 ** 31 - 1]
    pool.append(x, x, slots, F32)
    cache.append(x.astype(float), x.astype(float), slots)
    same_as(cache, pool, [0, 16])
    k, v = pool.read([-5, 0, 32, 2 ** 31 - 1, -2 ** 31])
    assert (k[[0, 2, 3, 4]] == -77).all() and (v[[0, 2, 3, 4]] == -77).all() and (k[1] != -77).all()
    assert pool.untouched()


def test_read_strides(dev, buf):
    step = Step(np.random.default_rng(2), 2, 64, [37], [0], F32)
    pool = pool_of(dev, buf, step)
    for ld in (128, 132, 260):
        k, v = pool.read(step.slots, ld)
        np.testing.assert_array_equal(k, step.cache.read(0, step.slots).astype(np.float32))
        np.testing.assert_array_equal(v, step.cache.read(1, step.slots).astype(np.float32))


# ---- tables and slots ------------------------------------------------------------------


def plan(block, lens, counts, tables, free, taken, rows):
    """The step's bookkeeping, one sequence after the other."""
    tables, new_lens, status = tables.copy(), lens.copy(), np.zeros(len(lens), np.int32)
    avail = len(free) - taken if 0 <= taken <= len(free) else 0
    start, used, granted, row_start = 0, 0, 0, []
    maps = np.full((3, rows), -1, np.int32)
    for i, (n, c) in enumerate(zip(lens.tolist(), counts.tolist())):
        row_start.append(min(start, rows))
        if n < 0 or c < 0:
            status[i] = 4
            continue
        end = start + c
        have, want = -(-n // block), -(-(n + c) // block)
        if want > tables.shape[1] or n + c > 2 ** 31 - 1:
            status[i] = 2
        elif end > rows:
            status[i], used = 3, used + want - have
        else:
            used += want - have
            if want > have and used > avail:
                status[i] = 1
        if status[i] == 0:
            if want > have:
                tables[i, have:want] = free[taken + used - (want - have):taken + used]
                granted = used
            new_lens[i] = n + c
            p = np.arange(n, n + c)
            page = tables[i, p // block]
            for m, x in zip(maps, (i, p, np.where(page < 0, -1, page * block + p % block))):
                m[start:end] = x
        start = end
    row_start.append(min(start, rows))
    return tables, new_lens, np.int32([taken + granted]), np.int32(row_start), *maps, status


def tables_case(rng, nseq, block, width, rows, n_free, taken, mean, odd=True):
    lens = rng.integers(0, block * width, nseq).astype(np.int32)
    counts = np.minimum(rng.geometric(1 / mean, nseq) - (rng.random(nseq) < 0.3), 4 * mean).astype(np.int32)
    if odd and nseq > 3:
        lens[nseq // 2], counts[nseq // 3] = -3, -1
        lens[nseq // 4] = 2 ** 31 - 2
    tables = rng.integers(0, 1000, (nseq, width)).astype(np.int32)
    if odd and nseq > 3:
        tables[1] = -1
    free = rng.permutation(5000)[:n_free].astype(np.int32)
    return block, lens, counts, tables, free, taken, rows


TABLES = [(1, 16, 8, 40, 30, 0, 2), (1, 16, 8, 0, 0, 0, 1), (3, 16, 4, 30, 2, 0, 8), (64, 16, 20, 100, 60, 5, 1),
          (65, 16, 20, 64, 60, 0, 1), (1000, 16, 30, 1500, 900, 100, 2), (1030, 16, 30, 2048, 3000, 0, 3),
          (1030, 16, 30, 2049, 300, 7, 3), (2100, 16, 12, 9000, 4000, 0, 5), (40, 1, 100, 400, 500, 3, 9),
          (40, 7, 30, 400, 200, 0, 9), (17, 100, 5, 5000, 40, 0, 300), (5, 16, 8, 40, 30, 31, 2), (5, 16, 8, 40, 30, -1, 2)]


@pytest.mark.parametrize("nseq,block,width,rows,n_free,taken,mean", TABLES)
@pytest.mark.parametrize("in_place", [False, True])
def test_tables(dev, buf, nseq, block, width, rows, n_free, taken, mean, in_place):
    from pagoda_amd.kv8 import kv_tables_dev

    rng = np.random.default_rng(nseq * 31 + rows)
    case = tables_case(rng, nseq, block, width, rows, n_free, taken, mean)
    block, lens, counts, tables, free, taken, rows = case
    want = plan(*case)
    up = lambda a: buf.up(a if a.size else np.zeros(1, a.dtype))
    ins = [up(a) for a in (lens, counts, tables, free, np.int32([taken]))]
    outs = [np.full_like(a, 99) for a in want[1:]]
    ptrs = [up(a) for a in outs]
    if in_place:
        ptrs[0], ptrs[1] = ins[0], ins[4]
    for _ in range(1 if in_place else 2):  # the same call again gives the same
        kv_tables_dev(dev, block, nseq, ins[0], ins[1], ins[2], width, ins[3], n_free, ins[4], rows, *ptrs)
    got = [buf.down(ins[2], tables)] + [buf.down(p, a) for p, a in zip(ptrs, outs)]
    for name, g, w in zip(("tables", "new_lens", "taken", "row_start", "seq", "pos", "slots", "status"), got, want):
        np.testing.assert_array_equal(g, w, err_msg=name)


def test_tables_without_sequences(dev, buf):
    from pagoda_amd.kv8 import kv_tables_dev

    maps = [np.full(5, 9, np.int32) for _ in range(3)]
    ptrs = [buf.up(a) for a in maps]
    taken, new, start = buf.up(np.int32([3])), buf.up(np.int32([0])), buf.up(np.int32([7]))
    kv_tables_dev(dev, 16, 0, 0, 0, 0, 4, 0, 0, taken, 5, 0, new, start, *ptrs, 0)
    assert buf.down(start, np.int32([0]))[0] == 0 and buf.down(new, np.int32([0]))[0] == 3
    assert all((buf.down(p, a) == -1).all() for p, a in zip(ptrs, maps))


# ---- attention -------------------------------------------------------------------------


class Call:
    """Device arrays of a step's attention; results are checked inside their rows' stride."""

    def __init__(self, dev, buf, step, pool, heads, t, q, gate=None, more=8):
        self.dev, self.buf, self.step, self.pool, self.heads, self.t = dev, buf, step, pool, heads, t
        self.width = heads * step.cache.hd
        self.ld = self.width + more
        self.q = buf.up(strided(q, self.ld, q.dtype.type(3)))
        self.gate = buf.up(strided(gate, self.width + 16, gate.dtype.type(3))) if gate is not None else 0
        self.ints = [buf.up(a) for a in (step.row_start, step.lens, step.tables)]
        self.fresh = np.full((step.rows + 2, self.width + 2 * more), 5, q.dtype)
        self.out = buf.up(self.fresh)

    def args(self):
        return (self.heads, self.q, self.ld, self.t, len(self.step.lens), *self.ints, self.step.width, self.step.rows)

    def result(self):
        got = self.buf.down(self.out, self.fresh)
        assert (got[self.step.rows:] == 5).all() and (got[:, self.width:] == 5).all()
        return value(got[:self.step.rows, :self.width], self.t).reshape(self.step.rows, self.heads, -1)

    def attn(self, max_rows=None):
        p = self.pool.pool
        size = p.attn_ws_bytes(self.heads, len(self.step.lens), self.step.width, self.step.rows)
        ws = self.buf.up(np.full(max(size, 16), 0xFF, np.uint8))
        most = max(self.step.new) if max_rows is None else max_rows
        p.attn_dev(*self.args(), most, self.out, self.fresh.shape[1], ws, size, self.gate, self.width + 16)
        return self.result()

    def workspace(self, top):
        size = self.pool.pool.sparse_ws_bytes(self.heads, self.step.rows, self.step.width, top)
        return self.buf.up(np.full(max(size, 16), 0xFF, np.uint8)), size

    def select(self, top, sinks, recent):
        sel, count = np.full((self.step.rows, self.step.cache.kv, top), 77, np.int32), np.full((self.step.rows, self.step.cache.kv), 77, np.int32)
        ps, pc = self.buf.up(sel), self.buf.up(count)
        self.pool.pool.select_dev(*self.args(), top, sinks, recent, ps, pc, *self.workspace(top))
        return self.buf.down(ps, sel), self.buf.down(pc, count)

    def sparse(self, sel, count):
        self.pool.pool.attn_sparse_dev(*self.args(), sel.shape[2], self.buf.up(sel), self.buf.up(count), self.out,
                                       self.fresh.shape[1], *self.workspace(sel.shape[2]), self.gate, self.width + 16)
        return self.result()


def queries(rng, step, heads, t, gate=False, scale=1.0):
    (q, qv), (g, gv) = (typed(rng.normal(0, s, (max(step.rows, 1), heads * step.cache.hd)), t) for s in (scale, 3.0))
    shape = (-1, heads, step.cache.hd)
    return q, qv.reshape(shape), (g, gv.reshape(shape)) if gate else (None, None)


def check_attention(dev, buf, rng, step, heads, t, gate=False, scale=1.0, **kw):
    pool = pool_of(dev, buf, step)
    q, qv, (g, gv) = queries(rng, step, heads, t, gate, scale)
    call = Call(dev, buf, step, pool, heads, t, q, g)
    want, bound = kv8.attention(step, qv, t, heads, gv)
    got = call.attn(**kw)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], bound[bad][:5])
    return call, got


@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_attention_decode(dev, buf, t, heads, kv, hd):
    """One token a sequence, contexts from one position to several chunks, page ends on both sides."""
    rng = np.random.default_rng(heads + hd + t)
    ctx = [1, 2, 15, 16, 17, 33, 64, 250, 257, 700]
    check_attention(dev, buf, rng, Step(rng, kv, hd, ctx, [1] * len(ctx), t), heads, t, gate=heads != 14)


@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_attention_chunks(dev, buf, t, heads, kv, hd):
    """Verify chunks, prompts behind prefixes and whole prompts; sequences without rows between them."""
    rng = np.random.default_rng(heads + hd + t + 7)
    ctx, new = [5, 40, 300, 77, 19, 130, 64], [5, 4, 33, 0, 19, 70, 1]
    check_attention(dev, buf, rng, Step(rng, kv, hd, ctx, new, t), heads, t, gate=heads == 14)


@pytest.mark.parametrize("t,heads,kv,hd,ctx,new", [
    (F32, 24, 4, 256, [5003], [1]), (BF16, 14, 2, 64, [9001, 3, 2000], [1, 1, 2]), (F16, 28, 4, 128, [2500, 2500], [4, 1]),
    (F32, 14, 2, 64, [1700], [130]), (BF16, 24, 4, 256, [900, 1025], [200, 65]), (F16, 8, 8, 128, [600], [257])])
def test_attention_long(dev, buf, t, heads, kv, hd, ctx, new):
    rng = np.random.default_rng(ctx[0])
    check_attention(dev, buf, rng, Step(rng, kv, hd, ctx, new, t), heads, t)


@pytest.mark.parametrize("t,heads,kv,hd,ctx,new", [
    (F16, 24, 4, 256, [3977], [236]), (F32, 24, 4, 256, [7000], [30]), (BF16, 8, 4, 128, [4000, 150], [1500, 140]),
    (F32, 8, 8, 128, [4000, 90], [2200, 90]), (F32, 14, 2, 64, [4000, 2000], [1300, 17]),
    (BF16, 24, 8, 64, [4000, 4000], [1500, 1300]), (F32, 6, 2, 256, [5000, 700, 33], [2500, 600, 33])])
def test_attention_of_prompts_on_long_contexts(dev, buf, t, heads, kv, hd, ctx, new):
    """Contexts cut into as many chunks as run at once, into chunks of a fixed size, and into as few as balance: some
    rows of each sequence against the definition, its first and last among them."""
    rng = np.random.default_rng(ctx[0] + new[0] + hd)
    step = Step(rng, kv, hd, ctx, new, t)
    pool = pool_of(dev, buf, step)
    q, qv, (g, gv) = queries(rng, step, heads, t, True)
    rows = list(step.each_row())
    ends = np.cumsum([0] + new)
    some = sorted(set(rng.integers(0, step.rows, 25)) | set(ends[:-1]) | set(ends[1:] - 1))
    step.each_row = lambda: [rows[i] for i in some]
    want, bound = kv8.attention(step, qv, t, heads, gv)
    got = Call(dev, buf, step, pool, heads, t, q, g).attn()
    bad = ~(np.abs(got - want) <= bound)[some]
    assert not bad.any(), (np.argwhere(bad)[:5], got[some][bad][:5], want[some][bad][:5])
    assert np.isfinite(got).all()


@pytest.mark.parametrize("t,heads,kv,hd", [(F32, 14, 2, 64), (F16, 24, 4, 256), (BF16, 28, 4, 128), (F32, 40, 1, 64)])
@pytest.mark.parametrize("most", [3, 9, 18, 19, 21, 22])
def test_attention_of_chunks_of_many_sizes(dev, buf, t, heads, kv, hd, most):
    """Verify chunks of up to 4 tiles and past them, whose kernels differ, next to single rows and none."""
    rng = np.random.default_rng(most + hd)
    ctx = [most, 700, 150, 1, 333, 64]
    check_attention(dev, buf, rng, Step(rng, kv, hd, ctx, [most, most, 2, 1, 0, most // 2], t), heads, t, gate=hd == 64)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("max_rows", [0, 1, 7, 10 ** 6])
def test_any_bound_on_the_rows(dev, buf, t, max_rows):
    rng = np.random.default_rng(3)
    step = Step(rng, 2, 128, [90, 40, 400, 1], [50, 3, 9, 1], t)
    check_attention(dev, buf, rng, step, 12, t, max_rows=max_rows)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 30.0, 1e4])
@pytest.mark.parametrize("t", [F32, BF16])
def test_attention_of_large_and_small_scores(dev, buf, t, scale):
    """From flat softmaxes to ones that are all on one position."""
    rng = np.random.default_rng(int(scale * 10) % 1000)
    step = Step(rng, 2, 128, [70, 300], [2, 1], t)
    check_attention(dev, buf, rng, step, 4, t, scale=scale)


def test_values_of_very_different_pages(dev, buf):
    """Pages whose powers of two lie far apart: no page's values drown in rounding of another's."""
    rng = np.random.default_rng(8)
    step = Step(rng, 1, 64, [96], [1], F32)
    size = (2.0 ** np.repeat([60, -60, 100, -100, 0, 3], 16))[:, None]
    k, v = rng.normal(0, 1, (2, 96, 64))
    step.k_raw, step.v_raw = np.float32(k), np.float32(v * size)
    step.cache = kv8.Cache(step.cache.n, 1, 64)
    step.cache.append(step.k_raw.astype(float), step.v_raw.astype(float), step.slots)
    check_attention(dev, buf, rng, step, 2, F32)


@pytest.mark.parametrize("t", [F32, F16])
def test_rows_that_attend_nothing(dev, buf, t):
    """Empty contexts and more rows than positions give zeros; rows of no sequence are left."""
    rng = np.random.default_rng(4)
    step = Step(rng, 2, 64, [0, 3, 40, 0], [1, 8, 2, 3], t)
    pool = pool_of(dev, buf, step)
    q, qv, (g, gv) = queries(rng, step, 6, t, True)
    call = Call(dev, buf, step, pool, 6, t, q, g)
    want, bound = kv8.attention(step, qv, t, 6, gv)
    got = call.attn()
    assert (np.abs(got - want) <= bound).all()
    empty = [r for r, _, seen in step.each_row() if seen == 0]
    assert len(empty) == 9 and not got[empty].any()
    # rows before the first sequence and behind the last
    step.row_start = np.int32([2, 2, 5, 5, 7])
    step.new = [0, 3, 0, 2]
    step.ctx, step.lens = [0, 3, 40, 40], np.int32([0, 3, 40, 40])
    step.tables[3] = step.tables[2]
    call = Call(dev, buf, step, pool, 6, t, q, g)
    want, bound = kv8.attention(step, qv, t, 6, gv)
    got = call.attn()
    assert (np.abs(got - want) <= bound)[2:7].all()
    assert (got[:2] == value(np.full(1, 5, q.dtype), t)).all() and (got[7:] == value(np.full(1, 5, q.dtype), t)).all()


def test_lengths_past_the_table(dev, buf):
    """Positions that the table has no page for do not exist; negative lengths attend nothing."""
    rng = np.random.default_rng(5)
    step = Step(rng, 1, 64, [64, 32], [2, 1], F32, widen=0)
    pool = pool_of(dev, buf, step)
    q, qv, _ = queries(rng, step, 3, F32)
    step.lens = np.int32([1000, -5])
    got = Call(dev, buf, step, pool, 3, F32, q).attn()
    step.ctx, step.new = [65, 0], [2, 1]  # both rows see all 64 positions
    step.tables = np.concatenate([step.tables, step.tables[:, :1]], 1)
    want, bound = kv8.attention(step, qv, F32, 3)
    k, v = (step.cache.values(w)[step.tables[0, :4], 0].reshape(64, 64) for w in range(2))
    for row in range(2):
        for h in range(3):
            o, b = kv8.attend(qv[row, h], k, v, F32)
            assert (np.abs(got[row, h] - o) <= b + np.abs(o) * 2.0 ** -24).all()
    assert not got[2].any()


@pytest.mark.parametrize("t", [F32, BF16])
def test_nonfinite_entries_reach_only_rows_that_attend_them(dev, buf, t):
    rng = np.random.default_rng(6)
    heads, kv, hd = 6, 2, 64
    step = Step(rng, kv, hd, [50, 40], [12, 3], t)
    bad = {F32: np.float32(np.nan), BF16: np.uint16(0x7F80)}[t]
    step.k_raw[44, 70] = bad       # sequence 0, position 44, head 1
    step.v_raw[50 + 39, 3] = bad   # sequence 1, its last position, head 0
    step.cache = kv8.Cache(step.cache.n, kv, hd)
    step.cache.append(value(step.k_raw, t), value(step.v_raw, t), step.slots)
    pool = pool_of(dev, buf, step)
    q, qv, _ = queries(rng, step, heads, t)
    call = Call(dev, buf, step, pool, heads, t, q)
    got = call.attn()
    want, bound = kv8.attention(step, qv, t, heads)
    hit = np.isnan(want)
    assert hit.any() and np.array_equal(np.isnan(got), hit)
    assert (np.abs(got - want) <= bound)[~hit].all()
    assert hit[6:12, 3:].all() and not hit[:6].any() and not hit[:12, :3].any() and hit[14, :3].all() and not hit[12:14].any()


def test_nonfinite_queries_stay_in_their_head(dev, buf):
    rng = np.random.default_rng(7)
    step = Step(rng, 2, 64, [50, 400], [3, 1], F32)
    pool = pool_of(dev, buf, step)
    q, qv, _ = queries(rng, step, 6, F32)
    q[1, 2 * 64 + 5], q[3, 5 * 64] = np.inf, np.nan
    got = Call(dev, buf, step, pool, 6, F32, q).attn()
    clean = np.ones((4, 6), bool)
    clean[1, 2] = clean[3, 5] = False
    want, bound = kv8.attention(step, np.where(np.isfinite(q), q, 0.0).astype(float).reshape(4, 6, 64), F32, 6)
    assert (np.abs(got - want) <= bound)[clean].all() and np.isnan(got[~clean]).all()


@pytest.mark.parametrize("t", [F32, F16])
def test_pages_outside_the_pool(dev, buf, t):
    """What attends them is NaN, and nothing else."""
    rng = np.random.default_rng(9)
    step = Step(rng, 2, 64, [60, 300, 20], [20, 1, 1], t)
    pool = pool_of(dev, buf, step)
    q, qv, _ = queries(rng, step, 4, t)
    want, bound = kv8.attention(step, qv, t, 4)
    step.tables[0, 3], step.tables[1, 7] = step.cache.n, -1  # positions 48.. of sequence 0
    got = Call(dev, buf, step, pool, 4, t, q).attn()
    bad = np.zeros(22, bool)
    bad[8:21] = True
    assert np.isnan(got[bad]).all() and (np.abs(got - want) <= bound)[~bad].all()
    for page in (2 ** 31 - 1, -2 ** 31, 1 << 27):
        step.tables[2, 0] = page
        assert np.isnan(Call(dev, buf, step, pool, 4, t, q).attn()[21]).all()


def test_the_same_call_gives_the_same_bits(dev, buf):
    rng = np.random.default_rng(10)
    for t, ctx, new in ((F32, [3000, 17, 900], [1, 1, 1]), (BF16, [500, 90], [200, 40])):
        call, got = check_attention(dev, buf, rng, Step(rng, 2, 128, ctx, new, t), 14, t)
        for _ in range(3):
            assert np.array_equal(call.attn(), got)


def test_many_sequences(dev, buf):
    """More sequences than lanes of a wave, some without rows."""
    rng = np.random.default_rng(11)
    n = 150
    new = rng.integers(0, 3, n)
    step = Step(rng, 1, 64, np.maximum(rng.integers(0, 90, n), new).tolist(), new.tolist(), F32)
    check_attention(dev, buf, rng, step, 2, F32)


# ---- selection and attention over it -------------------------------------------------------


@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_select_and_attend(dev, buf, t, heads, kv, hd):
    rng = np.random.default_rng(heads + hd + t + 20)
    ctx, new = [900, 1, 17, 160, 0, 333, 2100], [1, 1, 2, 0, 1, 3, 1]
    step = Step(rng, kv, hd, ctx, new, t)
    pool = pool_of(dev, buf, step)
    q, qv, (g, gv) = queries(rng, step, heads, t, gate=heads != 4)
    call = Call(dev, buf, step, pool, heads, t, q, g)
    for top, sinks, recent in ((9, 1, 2), (20, 0, 0), (200, 3, 1)):
        want = kv8.select(step, qv, heads, top, sinks, recent)
        sel, count = call.select(top, sinks, recent)
        for row in range(step.rows):
            for h in range(kv):
                w = want[row][h]
                assert count[row, h] == len(w) and sel[row, h].tolist() == w + [-1] * (top - len(w)), (row, h)
        out, bound = kv8.attention(step, qv, t, heads, gv, want)
        got = call.sparse(sel, count)
        assert (np.abs(got - out) <= bound).all()
        assert np.array_equal(call.sparse(sel, count), got)


def test_selection_of_everything_is_attention(dev, buf):
    rng = np.random.default_rng(30)
    step = Step(rng, 2, 64, [700, 90], [1, 3], F32)
    call, dense = check_attention(dev, buf, rng, step, 8, F32)
    sel, count = call.select(step.width, 0, 1)
    assert (count == [[44, 44], [6, 6], [6, 6], [6, 6]]).all()
    assert np.abs(call.sparse(sel, count) - dense).max() < 1e-5 * np.abs(dense).max()


def test_ties_go_to_the_lower_page(dev, buf):
    """Pages of equal keys, some of them twice as large: by score, then by place."""
    rng = np.random.default_rng(31)
    step = Step(rng, 1, 64, [320], [1], F32)
    page = rng.normal(0, 1, (16, 64)).astype(np.float32)
    times = np.where(np.isin(np.arange(20), (3, 11, 12, 17)), 2.0, 1.0).astype(np.float32)
    step.k_raw = (page[None] * times[:, None, None]).reshape(320, 64)
    step.cache = kv8.Cache(step.cache.n, 1, 64)
    step.cache.append(step.k_raw.astype(float), value(step.v_raw, F32), step.slots)
    pool = pool_of(dev, buf, step)
    q, qv, _ = queries(rng, step, 3, F32)
    q[:] = np.abs(q)
    page_sum = lambda s: [p for p in range(20) if times[p] == s]
    qv = q.astype(float).reshape(1, 3, 64)
    call = Call(dev, buf, step, pool, 3, F32, q)
    for top in (2, 4, 7, 19):
        sel, count = call.select(top, 0, 0)
        assert count[0, 0] == top
        assert sel[0, 0].tolist() == sorted((page_sum(2.0) + page_sum(1.0))[:top])
        assert kv8.select(step, qv, 3, top, 0, 0)[0][0] == sel[0, 0].tolist()
    q[:] = 0  # all scores are zero, of both signs
    assert Call(dev, buf, step, pool, 3, F32, q).select(5, 0, 2)[0][0, 0].tolist() == [0, 1, 2, 18, 19]


def test_selection_past_bad_input(dev, buf):
    """Pages outside the pool score lowest; non-finite entries of q count as zero."""
    rng = np.random.default_rng(32)
    step = Step(rng, 2, 64, [500, 800], [1, 2], F32)
    pool = pool_of(dev, buf, step)
    q, qv, _ = queries(rng, step, 4, F32)
    q[0, 7], q[2, 100], q[2, 130] = np.inf, np.nan, -np.inf
    step.tables[0, [2, 30]], step.tables[1, 5] = [step.cache.n, -4], 2 ** 31 - 1
    qv = q.astype(float).reshape(3, 4, 64)
    call = Call(dev, buf, step, pool, 4, F32, q)
    for top in (4, 31):
        want = kv8.select(step, qv, 4, top, 1, 1)
        sel, count = call.select(top, 1, 1)
        for row in range(3):
            for h in range(2):
                assert sel[row, h, :count[row, h]].tolist() == want[row][h]


def test_scores_past_the_largest_f32(dev, buf):
    """Key exponents up to the largest: scores that overflow are equal, and forced pages come before them."""
    rng = np.random.default_rng(33)
    step = Step(rng, 1, 64, [160], [1], F32)
    step.k_raw = (rng.normal(0, 1, (160, 64)) * 2.0 ** np.repeat([100, 118, 0, 120, 119, 3, 118, 60, 2, 1], 16)[:, None]).astype(np.float32)
    step.cache = kv8.Cache(step.cache.n, 1, 64)
    step.cache.append(step.k_raw.astype(float), value(step.v_raw, F32), step.slots)
    pool = pool_of(dev, buf, step)
    q, qv, _ = queries(rng, step, 2, F32)
    for top in (1, 2, 3, 5):
        sel, _ = Call(dev, buf, step, pool, 2, F32, q).select(top, 0, 1)
        assert sel[0, 0].tolist() == kv8.select(step, qv, 2, top, 0, 1)[0][0]


@pytest.mark.parametrize("t,heads,kv,hd", [(F32, 6, 2, 64), (BF16, 20, 1, 128), (F16, 3, 3, 256)])
def test_lists_of_ones_own(dev, buf, t, heads, kv, hd):
    """Any order, entries outside the table skipped, a page named twice counted twice, empty lists."""
    rng = np.random.default_rng(34 + hd)
    step = Step(rng, kv, hd, [300, 70], [2, 1], t)
    pool = pool_of(dev, buf, step)
    q, qv, _ = queries(rng, step, heads, t)
    call = Call(dev, buf, step, pool, heads, t, q)
    top = 90
    sel = np.full((3, kv, top), 10 ** 6, np.int32)
    count = np.zeros((3, kv), np.int32)
    picked = {r: [] for r in range(3)}
    for r in range(3):
        for h in range(kv):
            n = [top + 50, 11, 0][(r + h) % 3]
            p = rng.integers(0, 19 if r < 2 else 5, min(n, top))
            count[r, h] = n
            sel[r, h, :len(p)] = p
            junk = rng.random(len(p)) < 0.2
            sel[r, h, :len(p)][junk] = rng.choice([-1, -9, step.width, 2 ** 30], junk.sum())
            picked[r].append(p[~junk])
    want, bound = kv8.attention(step, qv, t, heads, picked=picked)
    got = call.sparse(sel, count)
    assert (np.abs(got - want) <= bound).all()
    count[:] = -3
    assert not call.sparse(sel, count).any()


def test_selection_of_many_equal_scores(dev, buf):
    """More pages of one score than are settled by rank, above and below others, past what threads hold of
    keys: the lowest ones that fit."""
    from pagoda_amd import Kv8Pool
    from pagoda_amd.kv8 import page_bytes

    rng = np.random.default_rng(35)
    for pages, distinct in ((1500, 1), (3000, 3), (9100, 2), (9100, 5000), (20000, 40)):
        # `distinct` pages of keys, named by the table many times over
        d = min(distinct, 600)
        k = np.repeat(rng.normal(0, 1, (d, 1, 64)), 16, 1).reshape(-1, 64).astype(np.float32)
        slots = np.arange(16 * d, dtype=np.int32)
        cache = kv8.Cache(d, 1, 64)
        cache.append(k.astype(float), k.astype(float), slots)
        pool = GpuPool(dev, buf, 1, 64, d)
        pool.append(k, k, slots, F32)
        table = rng.integers(0, d, pages).astype(np.int32)
        q = rng.normal(0, 1, (1, 64)).astype(np.float32)
        q8 = np.rint(q[0].astype(float) * 2.0 ** -kv8.holds(np.abs(q).max(), 127.0))
        by_page = []
        for p in range(d):
            hi, lo = (b[0] for b in cache.bounds(p))
            by_page.append(np.maximum(q8 * hi, q8 * lo).sum() * 2.0 ** cache.exps[0, p, 0])
        score = np.array(by_page)[table]
        ptrs = [buf.up(a) for a in (q, np.int32([0, 1]), np.int32([pages * 16]), table)]
        for top, sinks, recent in ((1, 0, 0), (700, 0, 0), (1400, 5, 3), (pages - 1, 0, 1), (pages, 0, 0)):
            sel, count = np.full(top, 9, np.int32), np.int32([9])
            ps, pc = buf.up(sel), buf.up(count)
            size = pool.pool.sparse_ws_bytes(1, 1, pages, top)
            pool.pool.select_dev(1, ptrs[0], 64, F32, 1, *ptrs[1:], pages, 1, top, sinks, recent, ps, pc,
                                 buf.up(np.zeros(size, np.uint8)), size)
            forced = (np.arange(pages) < sinks) | (np.arange(pages) >= pages - recent)
            want = np.sort(np.lexsort((np.arange(pages), -score, ~forced))[:top])
            assert buf.down(pc, count)[0] == top
            np.testing.assert_array_equal(buf.down(ps, sel), want, err_msg=str((pages, distinct, top)))


@pytest.mark.parametrize("kv,hd", [(1, 64), (3, 128), (2, 256)])
def test_read_of_many_rows(dev, buf, kv, hd):
    """More rows than the call reads one by one (2047): whole sequences, any order, runs across pages, slots
    twice and outside the pool."""
    rng = np.random.default_rng(40 + hd)
    step = Step(rng, kv, hd, [400, 77, 5], [0, 0, 0], F32)
    pool = pool_of(dev, buf, step)
    same_as(step.cache, pool, step.slots)
    some = np.concatenate([step.slots[3:200], rng.permutation(step.slots), step.slots[::-1][:100], np.repeat(step.slots[7], 19)] * 6)
    assert len(some) > 4096
    same_as(step.cache, pool, some)
    bad = rng.random(len(some)) < 0.2
    some[bad] = rng.choice([-1, -2, -3, step.cache.n * 16, 2 ** 31 - 1, -2 ** 31], bad.sum())
    k, v = pool.read(some, kv * hd + 4)
    assert (k[bad] == -77).all() and (v[bad] == -77).all()
    for got, w in ((k, 0), (v, 1)):
        np.testing.assert_array_equal(got[~bad], step.cache.read(w, some[~bad]).astype(np.float32))


@pytest.mark.parametrize("t,kv,hd", [(F32, 1, 64), (F16, 2, 128), (BF16, 1, 256)])
@pytest.mark.parametrize("rows", [255, 256, 257, 1000, 2047, 2048, 2049, 5000])
def test_write_of_many_rows(dev, buf, t, kv, hd, rows):
    """Calls of sizes that are shared out to workgroups and read in different ways: runs of one to many pages that
    begin and end anywhere, single rows, and rows of no slot between them; then the pages' second halves."""
    rng = np.random.default_rng(rows + hd)
    slots, ends, page = [], [], 0
    numbers = rng.permutation(rows + 8)
    while len(slots) < rows:
        kind = rng.integers(4)
        if kind == 0:
            slots += [-1, 2 ** 31 - 1, (rows + 8) * PAGE][: rng.integers(1, 4)]
            continue
        n = min(1 if kind == 1 else rng.integers(1, 17) if kind == 2 else rng.integers(17, 200), rows - len(slots))
        if n <= 0:
            break
        place = np.arange(n)
        slots += list(numbers[page + place // PAGE] * PAGE + place % PAGE)
        page += -(-n // PAGE)
        ends.append(slots[-1])
    slots = np.array(slots[:rows])
    cache, pool = kv8.Cache(rows + 8, kv, hd), GpuPool(dev, buf, kv, hd, rows + 8)
    for _ in range(2):
        size = 2.0 ** rng.integers(-12, 6, (2, len(slots), 1)) * rng.normal(0, 1, (2, len(slots), kv * hd))
        (kr, k), (vr, v) = typed(size[0], t), typed(size[1], t)
        pool.append(kr, vr, slots, t, kv * hd + 8, kv * hd)
        cache.append(k, v, slots)
        live = slots[(slots >= 0) & (slots < cache.n * PAGE)]
        same_as(cache, pool, live)
        # (go on behind the last rows of the runs, to their pages' ends)
        slots = np.array([s for e in ends for s in range(e + 1, (e | (PAGE - 1)) + 1)], np.int64)
    assert pool.untouched()


@pytest.mark.parametrize("t,heads,kv,hd", [(F32, 14, 2, 64), (F16, 28, 4, 128), (BF16, 24, 4, 256), (F32, 17, 1, 64)])
def test_selection_through_tables_of_any_width(dev, buf, t, heads, kv, hd):
    """The pages do not hang on the width of the tables, which the scores are split by, nor on the size of a group."""
    rng = np.random.default_rng(50 + hd)
    step = Step(rng, kv, hd, [1000, 40, 530], [1, 2, 1], t)
    pool = pool_of(dev, buf, step)
    q, qv, _ = queries(rng, step, heads, t)
    narrow = step.tables
    for top, sinks, recent in ((5, 0, 0), (30, 1, 2)):
        want = kv8.select(step, qv, heads, top, sinks, recent)
        for width in (64, 1024, 1025, 5000):
            step.tables = np.full((3, width), -1, np.int32)
            step.tables[:, :min(width, narrow.shape[1])] = narrow[:, :width]
            step.width = width
            sel, count = Call(dev, buf, step, pool, heads, t, q).select(top, sinks, recent)
            for row in range(step.rows):
                for h in range(kv):
                    assert sel[row, h].tolist() == want[row][h] + [-1] * (top - len(want[row][h])), (width, row, h)
        step.tables, step.width = narrow, narrow.shape[1]


def test_rows_end_where_the_call_says(dev, buf):
    """Row starts past the number of rows: the rows that are there are their sequence's latest, to every call."""
    rng = np.random.default_rng(60)
    step = Step(rng, 1, 64, [200, 90], [2, 3], F32)
    pool = pool_of(dev, buf, step)
    q, qv, _ = queries(rng, step, 2, F32)
    step.row_start = np.int32([0, 2, 9])
    call = Call(dev, buf, step, pool, 2, F32, q)
    want, bound = kv8.attention(step, qv, F32, 2)
    assert (np.abs(call.attn() - want) <= bound).all()
    sel, count = call.select(step.width, 0, 0)
    assert count[:, 0].tolist() == [13, 13, 6, 6, 6]
    assert (np.abs(call.sparse(sel, count) - want) <= bound).all()
