"""The 8-bit KV cache as callers launch it: a server's steps from the bookkeeping to the attention, beside the
f32 attention, in HIP graphs, on several handles and threads, with offsets past 32 bits."""
import ctypes as C
import threading

import numpy as np
import pytest

import kv8
from kv8 import BF16, F16, F32, PAGE, Step, typed, value
from test_gpu_kv8 import Call, GpuPool, check_attention, pool_of, queries
from test_gpu_mxfp4 import Buffers, buf  # noqa: F401
from test_gpu_mxfp4_launches import Graph

pytestmark = pytest.mark.gpu


class Server:
    """Device arrays of a fixed number of sequences and rows; host copies follow the definition."""

    def __init__(self, dev, buf, nseq, rows, kv, hd, heads, t, n_pages, width, top=0):
        from pagoda_amd import Kv8Pool

        self.dev, self.buf, self.t, self.heads, self.kv, self.hd = dev, buf, t, heads, kv, hd
        self.nseq, self.rows, self.width, self.top = nseq, rows, width, top
        self.cache = kv8.Cache(n_pages, kv, hd)
        self.pool = GpuPool(dev, buf, kv, hd, n_pages)
        rng = np.random.default_rng(nseq + rows)
        self.free = rng.permutation(n_pages).astype(np.int32)
        self.lens, self.tables, self.taken = np.zeros(nseq, np.int32), np.full((nseq, width), -1, np.int32), 0
        ints = lambda *s: buf.up(np.full(s, 1234567, np.int32))
        self.p = dict(lens=buf.up(self.lens), tables=buf.up(self.tables), taken=buf.up(np.int32([0])), free=buf.up(self.free),
                      counts=ints(nseq), row_start=ints(nseq + 1), seq=ints(rows), pos=ints(rows), slots=ints(rows),
                      status=ints(nseq))
        dtype = {F32: np.float32, F16: np.float16, BF16: np.uint16}[t]
        zeros = lambda w: buf.up(np.zeros((rows, w), dtype))
        self.p.update(k=zeros(kv * hd), v=zeros(kv * hd), q=zeros(heads * hd), out=zeros(heads * hd))
        self.empty = np.zeros((rows, heads * hd), dtype)
        self.size = max(self.pool.pool.attn_ws_bytes(heads, nseq, width, rows),
                        self.pool.pool.sparse_ws_bytes(heads, rows, width, top) if top else 0)
        self.ws = buf.up(np.full(max(self.size, 16), 0xFF, np.uint8))
        if top:
            self.p.update(sel=ints(rows, kv, top), count=ints(rows, kv), sparse=zeros(heads * hd))

    def put(self, ptr, a):
        from pagoda_amd._lib import call

        a = np.ascontiguousarray(a)
        call("pgd_device_memcpy", self.dev.handle, C.c_void_p(ptr), a.ctypes.data_as(C.c_void_p), C.c_size_t(a.nbytes), 0)

    def calls(self):
        """A step, all from device memory: lengths and the pages taken move on in place."""
        from pagoda_amd.kv8 import kv_tables_dev

        p, w = self.p, self.kv * self.hd
        kv_tables_dev(self.dev, PAGE, self.nseq, p["lens"], p["counts"], p["tables"], self.width, p["free"], len(self.free),
                      p["taken"], self.rows, p["lens"], p["taken"], p["row_start"], p["seq"], p["pos"], p["slots"], p["status"])
        self.pool.pool.append_dev(p["k"], w, p["v"], w, self.t, p["slots"], self.rows)
        args = (self.heads, p["q"], self.heads * self.hd, self.t, self.nseq, p["row_start"], p["lens"], p["tables"],
                self.width, self.rows)
        self.pool.pool.attn_dev(*args, self.rows, p["out"], self.heads * self.hd, self.ws, self.size)
        if self.top:
            self.pool.pool.select_dev(*args, self.top, 1, 1, p["sel"], p["count"], self.ws, self.size)
            self.pool.pool.attn_sparse_dev(*args, self.top, p["sel"], p["count"], p["sparse"], self.heads * self.hd, self.ws,
                                           self.size)

    def step(self, rng, counts, run):
        """Feeds counts rows, runs the step, checks it against the definition."""
        n = int(np.sum(counts))
        rows = lambda w: typed(rng.normal(0, 1, (self.rows, w)), self.t)
        (k, kvv), (v, vv), (q, qv) = rows(self.kv * self.hd), rows(self.kv * self.hd), rows(self.heads * self.hd)
        for name, a in (("counts", np.int32(counts)), ("k", k), ("v", v), ("q", q), ("out", self.empty)):
            self.put(self.p[name], a)
        run()
        step = Step.__new__(Step)
        step.new, step.cache, step.t, step.width, slots = list(counts), self.cache, self.t, self.width, []
        for s, c in enumerate(counts):
            for p in range(self.lens[s], self.lens[s] + c):
                if p % PAGE == 0:
                    self.tables[s, p // PAGE] = self.free[self.taken]
                    self.taken += 1
                slots.append(self.tables[s, p // PAGE] * PAGE + p % PAGE)
            self.lens[s] += c
        step.ctx, step.lens, step.tables, step.rows = self.lens.tolist(), self.lens, self.tables, n
        step.row_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.cache.append(kvv[:n], vv[:n], slots)
        down = lambda name, a: self.buf.down(self.p[name], a)
        assert np.array_equal(down("lens", self.lens), self.lens) and np.array_equal(down("tables", self.tables), self.tables)
        assert down("taken", np.int32([0]))[0] == self.taken and not down("status", self.lens).any()
        assert np.array_equal(down("slots", np.zeros(self.rows, np.int32)), slots + [-1] * (self.rows - n))
        want, bound = kv8.attention(step, qv.reshape(self.rows, self.heads, -1), self.t, self.heads)
        got = down("out", self.empty)
        assert not got[n:].any()
        got = value(got[:n], self.t).reshape(want.shape)
        assert (np.abs(got - want) <= bound).all()
        if self.top:
            picked = kv8.select(step, qv.reshape(self.rows, self.heads, -1), self.heads, self.top, 1, 1)
            sel = down("sel", np.zeros((self.rows, self.kv, self.top), np.int32))
            for row in range(n):
                for h in range(self.kv):
                    assert sel[row, h, :len(picked[row][h])].tolist() == picked[row][h]
            want, bound = kv8.attention(step, qv.reshape(self.rows, self.heads, -1), self.t, self.heads, None, picked)
            assert (np.abs(value(down("sparse", self.empty)[:n], self.t).reshape(want.shape) - want) <= bound).all()


@pytest.mark.parametrize("t,kv,hd,heads,top", [(F32, 2, 64, 6, 0), (BF16, 4, 128, 28, 3), (F16, 1, 256, 6, 4)])
def test_a_server_steps(dev, buf, t, kv, hd, heads, top):
    """Prompts, decode and verify rows over changing sequences, with rows to spare."""
    rng = np.random.default_rng(hd)
    s = Server(dev, buf, 4, 60, kv, hd, heads, t, 40, 9, top)
    for counts in ((40, 0, 3, 1), (1, 30, 1, 0), (1, 1, 1, 1), (4, 4, 0, 4), (0, 0, 0, 0), (1, 1, 50, 1), (1, 1, 1, 1)):
        s.step(rng, counts, s.calls)


def test_a_captured_step_replays(dev, buf):
    """Two servers' steps in a graph each, replayed in turn while lengths grow and eager calls run
    between them: every replay is a step as it would run eagerly."""
    rng = np.random.default_rng(77)
    a = Server(dev, buf, 3, 12, 2, 64, 6, F32, 40, 12, 3)
    b = Server(dev, buf, 2, 40, 1, 128, 4, BF16, 40, 20, 4)
    a.step(rng, (5, 0, 7), a.calls)
    b.step(rng, (30, 9), b.calls)
    graphs = [Graph(dev, s.calls) for s in (a, b)]
    try:
        for counts_a, counts_b in (((1, 1, 1), (1, 1)), ((4, 4, 4), (38, 2)), ((0, 10, 1), (1, 4)), ((1, 1, 1), (40, 0)),
                                   ((1, 0, 9), (1, 1))):
            a.step(rng, counts_a, graphs[0].replay)
            b.step(rng, counts_b, graphs[1].replay)
            step = Step(rng, 2, 64, [90], [3], F16)
            check_attention(dev, buf, rng, step, 4, F16)  # (eager, with memory of its own)
    finally:
        dev.sync()
        for g in graphs:
            g.close()


def test_maps_serve_the_f32_attention_too(dev, buf):
    """seq_of_row, pos_of_row and tables of a step, taken by pgd_attn_decode_dev over f32 pages."""
    from pagoda_amd._lib import call
    from pagoda_amd.kv8 import kv_tables_dev

    rng = np.random.default_rng(5)
    lens, counts, width, heads, kv, hd = np.int32([20, 0, 47]), np.int32([1, 5, 2]), 4, 4, 2, 64
    tables, free = np.full((3, width), -1, np.int32), np.int32([9, 2, 7, 1])
    tables[0, :2], tables[2, :3] = [3, 4], [0, 5, 6]
    up = buf.up
    pl, pc, pt, pf, pk = map(up, (lens, counts, tables, free, np.int32([0])))
    rows = 8
    outs = [up(np.zeros(n, np.int32)) for n in (3, 1, 4, rows, rows, rows, 3)]
    kv_tables_dev(dev, 16, 3, pl, pc, pt, width, pf, 4, pk, rows, *outs)
    after = buf.down(pt, tables)
    assert after[1, 0] == 9 and after[2, 3] == 2
    k, v = rng.normal(0, 1, (2, 10, kv, 16, hd)).astype(np.float32)
    q = rng.normal(0, 1, (rows, heads, hd)).astype(np.float32)
    out = np.zeros_like(q)
    po = up(out)
    call("pgd_attn_decode_dev", dev.handle, heads, kv, hd, 16, C.c_void_p(up(q)), None, C.c_void_p(up(k)), C.c_void_p(up(v)),
         C.c_void_p(outs[3]), C.c_void_p(outs[4]), C.c_void_p(pt), width, rows, C.c_void_p(po))
    got = buf.down(po, out)
    row = 0
    for s in range(3):
        for pos in range(lens[s], lens[s] + counts[s]):
            for h in range(heads):
                kk, vv = (x[after[s, :pos // 16 + 1], h // 2].reshape(-1, hd)[:pos + 1].astype(float) for x in (k, v))
                want, bound = kv8.attend(q[row, h].astype(float), kk, vv, F32)
                assert (np.abs(got[row, h] - want) <= bound + np.abs(want) * 2.0 ** -23).all()
            row += 1


def test_a_copied_page_is_the_page(dev, buf):
    """Copy on write: a page's bytes moved to another page, then written on by itself."""
    from pagoda_amd._lib import call

    rng = np.random.default_rng(6)
    cache, pool = kv8.Cache(4, 2, 128), GpuPool(dev, buf, 2, 128, 4)
    (kr, k), (vr, v) = (typed(rng.normal(0, 1, (12, 256)), F16) for _ in range(2))
    pool.append(kr[:9], vr[:9], np.arange(16, 25), F16)
    cache.append(k[:9], v[:9], np.arange(16, 25))
    size = pool.pool.page_bytes
    call("pgd_device_copy_dev", dev.handle, C.c_void_p(pool.at + 3 * size), C.c_void_p(pool.at + size), C.c_size_t(size))
    for array in (cache.units, cache.exps):
        array[:, 3] = array[:, 1]
    cache.filled[3] = 9
    pool.append(kr[9:], vr[9:], [57, 58, 59], F16)
    cache.append(k[9:], v[9:], [57, 58, 59])
    for s in (np.arange(16, 25), np.arange(48, 60)):
        for got, w in zip(pool.read(s), range(2)):
            np.testing.assert_array_equal(got, cache.read(w, s).astype(np.float32))


def test_offsets_past_32_bits(dev, buf):
    """Pages beyond 4 GiB of the pool, and of each other."""
    from pagoda_amd import Kv8Pool

    rng = np.random.default_rng(7)
    n = (5 << 30) // 35072
    big = Kv8Pool(dev, 4, 256, n)
    try:
        step = Step(rng, 4, 256, [200, 31], [3, 1], F32, spare=0)
        far = np.linspace(0, n - 1, step.cache.n).astype(np.int64)
        tables = np.where(step.tables >= 0, far[np.maximum(step.tables, 0)], -1).astype(np.int32)
        slots = (far[step.slots // 16] * 16 + step.slots % 16).astype(np.int32)
        assert int(slots.max()) // 16 * 35072 > 1 << 32
        up = buf.up
        big.append_dev(up(step.k_raw), 1024, up(step.v_raw), 1024, F32, up(slots), len(slots))
        k = np.zeros((len(slots), 1024), np.float32)
        pk, pv = up(k), up(k)
        big.read_dev(up(slots), len(slots), pk, 1024, pv, 1024)
        np.testing.assert_array_equal(buf.down(pk, k), step.cache.read(0, step.slots).astype(np.float32))
        q, qv, _ = queries(rng, step, 24, F32)
        pool = GpuPool.__new__(GpuPool)
        pool.pool = big
        call = Call(dev, buf, step, pool, 24, F32, q)
        call.ints[2] = up(tables)
        want, bound = kv8.attention(step, qv, F32, 24)
        assert (np.abs(call.attn() - want) <= bound).all()
        sel, count = call.select(5, 1, 1)
        picked = kv8.select(step, qv, 24, 5, 1, 1)
        assert all(sel[r, h].tolist() == picked[r][h] + [-1] * (5 - len(picked[r][h])) for r in range(4) for h in range(4))
        want, bound = kv8.attention(step, qv, F32, 24, None, picked)
        assert (np.abs(call.sparse(sel, count) - want) <= bound).all()
    finally:
        dev.sync()
        big.free()


def test_handles_and_threads(dev):
    """Two handles on the device, and two threads on each: calls with memory of their own do not meet."""
    from pagoda_amd import Device

    failed = []

    def work(d, seed):
        try:
            b = Buffers(d)
            try:
                rng = np.random.default_rng(seed)
                for ctx, new in (([300, 40], [1, 1]), ([60, 90], [30, 4]), ([700], [1])):
                    check_attention(d, b, rng, Step(rng, 2, 64, ctx, new, F32), 6, F32)
            finally:
                b.close()
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    other = Device("hip")
    threads = [threading.Thread(target=work, args=(d, i)) for i, d in enumerate((dev, other, dev, other))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    other.sync()
    other.close()
    assert not failed, failed


def test_the_callers_device_stays(dev, buf):
    """A call leaves the calling thread's current device as it was."""
    from pagoda_amd import lib

    now = C.c_int(-1)
    assert lib().hipGetDevice(C.byref(now)) == 0
    rng = np.random.default_rng(8)
    check_attention(dev, buf, rng, Step(rng, 1, 64, [40], [1], F32), 2, F32)
    after = C.c_int(-1)
    assert lib().hipGetDevice(C.byref(after)) == 0 and now.value == after.value
