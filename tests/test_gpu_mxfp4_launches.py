"""MXFP4 products as callers launch them: every block shape of the many-row kernel with
its ranges of k tiles, HIP graphs, several threads and handles, offsets past 32 bits."""
import ctypes as C
import threading

import numpy as np
import pytest

import mxfp4 as mx
from test_gpu_mxfp4 import BF16, F16, F32, Buffers, buf, matrix, pad16, run_planes, run_rows, weights  # noqa: F401

pytestmark = pytest.mark.gpu

PLANES = 3


def rows_and_values(rng, t, rows, k):
    """Activations of a type: what the call takes, and their values."""
    if t == PLANES:
        p = weights(rng, rows, k, spread=5)
        return p, mx.values(*p)
    raw, x = mx.rows_of(rng.normal(0, 1, (rows, k)).astype(np.float32), t)
    return raw, x.astype(np.float64)


def product(dev, buf, m, t, raw, **kw):
    return run_planes(dev, buf, m, raw, **kw) if t == PLANES else run_rows(dev, buf, m, raw, t, **kw)


# sizes estimated fastest with each block shape, once undivided and once in ranges of k tiles
LAUNCHES = [
    (PLANES, 5008, 160, 1300), (PLANES, 2000, 8224, 1100), (PLANES, 2000, 160, 1100), (PLANES, 1000, 6144, 1100),
    (PLANES, 1000, 160, 1100), (PLANES, 200, 4096, 1100), (PLANES, 2100, 160, 200), (PLANES, 200, 4096, 333),
    (F16, 2100, 160, 1100), (F16, 1000, 2080, 1100), (F32, 1000, 160, 1100), (BF16, 333, 4096, 600),
    (F32, 333, 160, 600), (F32, 48, 4096, 17), (F16, 333, 1024, 333), (BF16, 1000, 4096, 65),
    (F32, 1000, 512, 1100), (F32, 1000, 4096, 333), (F32, 200, 1024, 1100), (F32, 48, 4096, 600),
]


@pytest.mark.parametrize("t,n,k,rows", LAUNCHES)
def test_many_rows(dev, buf, t, n, k, rows):
    """Plain and with a residual; the same call again gives the same bits."""
    rng = np.random.default_rng(n + k + rows + t)
    w = weights(rng, n, k)
    raw, x = rows_and_values(rng, t, rows, k)
    m, wv = matrix(dev, w), mx.values(*w)
    want, bound = x @ wv.T, mx.product_bound(x, wv)
    got = product(dev, buf, m, t, raw, ldy_more=1)
    assert (np.abs(got - want) <= bound).all()
    for _ in range(3):
        assert np.array_equal(product(dev, buf, m, t, raw, ldy_more=1), got)
    res = rng.normal(0, 1, (rows, n)).astype(np.float32)
    got = product(dev, buf, m, t, raw, res=res)
    assert (np.abs(got - (res + want)) <= bound + 2.0 ** -23 * np.abs(res + want)).all()


@pytest.mark.parametrize("t,n,k,rows", [
    (PLANES, 5008, 160, 600), (PLANES, 1000, 8224, 1100), (PLANES, 1000, 160, 1100), (PLANES, 200, 6144, 2500),
    (PLANES, 1000, 160, 600), (PLANES, 200, 4096, 600), (PLANES, 2100, 160, 200), (PLANES, 200, 4096, 150),
    (F32, 1000, 160, 1100), (F32, 1000, 160, 600), (F32, 333, 160, 600), (F32, 48, 4096, 17),
    (F32, 1000, 512, 600), (F32, 333, 4096, 600), (F32, 333, 1024, 600), (F32, 333, 4096, 150),
])
def test_many_rows_of_a_pair(dev, buf, t, n, k, rows):
    rng = np.random.default_rng(n + k + rows + t + 1)
    g, u = weights(rng, n, k), weights(rng, n, k)
    raw, x = rows_and_values(rng, t, rows, k)
    gm, um, gv, uv = matrix(dev, g), matrix(dev, u), mx.values(*g), mx.values(*u)
    want = mx.silu(x @ gv.T) * (x @ uv.T)
    got = product(dev, buf, gm, t, raw, up=um)
    assert (np.abs(got - want) <= mx.swiglu_bound(x, gv, uv)).all()
    assert np.array_equal(product(dev, buf, gm, t, raw, up=um), got)
    same = product(dev, buf, gm, t, raw, up=gm)  # one matrix as both
    assert (np.abs(same - mx.silu(x @ gv.T) * (x @ gv.T)) <= mx.swiglu_bound(x, gv, gv)).all()


@pytest.mark.parametrize("rows", [17, 300])
def test_f32_rows_beside_an_outlier(dev, buf, rows):
    """Many f32 rows are held to 2^-30 of the power of two above their block's largest
    magnitude: the outlier's weights are zero, so all of the error is that rounding."""
    rng = np.random.default_rng(rows)
    n, k = 200, 1024
    codes, scales = weights(rng, n, k)
    codes[:, 0::16] &= 0xF0  # each block's first element
    x = rng.normal(0, 1, (rows, k)).astype(np.float32)
    x[:, 0::32] = (1.5 * 2.0 ** rng.integers(-30, 30, (rows, k // 32))).astype(np.float32)
    x[:, 32:64] *= np.float32(2.0 ** -60)
    wv, xd = mx.values(codes, scales), x.astype(np.float64)
    top = np.abs(xd).reshape(rows, -1, 32).max(-1)
    held = 2.0 ** (np.floor(np.log2(top)) + 1 - 30)
    live = np.where(np.arange(k) % 32 == 0, 0, xd)
    # (six digits' products a value instead of one, whose partial sums stay below twice the value)
    bound = 12 * mx.product_bound(live, wv) + held.repeat(32, 1) @ np.abs(wv).T
    got = run_rows(dev, buf, matrix(dev, (codes, scales)), x, F32)
    assert (np.abs(got - xd @ wv.T) <= bound).all()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 4, 12, 40, 300])
def test_values_below_the_normal_range(dev, buf, t, rows):
    """Subnormal activations under large weights, and weights of the smallest scales under large
    activations, one product per output: f32 rows past 16 are held to steps of 2^-130 (so within
    2^-131), fewer lose what is below 2^-133, the smallest bf16 number, which their last term
    (the truncation of what the others leave) cannot hold. bf16 rows lose nothing."""
    rng = np.random.default_rng(rows + t)
    n, k = 40, 256
    x = np.zeros((rows, k), np.float32)
    at = rng.integers(0, k, rows)
    x[np.arange(rows), at] = (rng.uniform(1, 2, rows) * 2.0 ** rng.integers(-140, -105, rows)).astype(np.float32)
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    for scale, rows_x in ((127 + 100, x), (0, np.where(x != 0, np.float32(1.25 * 2.0 ** 100), np.float32(0)))):
        w = codes, np.full((n, k // 32), scale, np.uint8)
        raw, xv = mx.rows_of(rows_x, t)
        wv, xd = mx.values(*w), xv.astype(np.float64)
        want = xd @ wv.T
        step = 0 if t == BF16 else 2.0 ** -131 if rows > 16 else 2.0 ** -133
        got = run_rows(dev, buf, matrix(dev, w), raw, t)
        assert (np.abs(got - want) <= 4 * 2.0 ** -23 * np.abs(want) + step * np.abs(wv[:, at].T)).all()


def test_residual_of_another_stride(dev, buf):
    rng = np.random.default_rng(12)
    n, k, ldres = 100, 160, 131
    w = weights(rng, n, k)
    m, wv = matrix(dev, w), mx.values(*w)
    for rows in (1, 30, 200):
        x, res = rng.normal(0, 1, (rows, k)).astype(np.float32), rng.normal(0, 1, (rows, ldres)).astype(np.float32)
        py = buf.up(np.zeros((rows, n), np.float32))
        m.gemv_dev(buf.up(x), k, rows, py, n, F32, buf.up(res), ldres)
        want = res[:, :n] + x.astype(np.float64) @ wv.T
        got = buf.down(py, np.zeros((rows, n), np.float32))
        assert (np.abs(got - want) <= mx.product_bound(x.astype(np.float64), wv) + 2.0 ** -23 * np.abs(want)).all()


def test_no_rows(dev, buf):
    """Nothing is written, and null rows are as good as any."""
    from pagoda_amd import Matrix
    from pagoda_amd.matrix import mxfp4_quantize_dev

    m = matrix(dev, weights(np.random.default_rng(1), 48, 96))
    y = np.full((2, 48), 55.0, np.float32)
    c, s = np.full((2, 48), 9, np.uint8), np.full((2, 16), 9, np.uint8)
    py, px, pc, ps = buf.up(y), buf.up(np.zeros((2, 96), np.float32)), buf.up(c), buf.up(s)
    for t in (F32, F16, BF16):
        m.gemv_dev(px, 96, 0, py, 48, t)
        mxfp4_quantize_dev(dev, px, t, 96, 0, 96, pc, 48, ps, 16)
    m.gemv_mx_dev(pc, 48, ps, 16, 0, py, 48)
    Matrix.gemv_swiglu_dev(m, m, px, 96, 0, py, 48)
    Matrix.gemv_swiglu_mx_dev(m, m, pc, 48, ps, 16, 0, py, 48)
    assert np.array_equal(buf.down(py, y), y) and np.array_equal(buf.down(pc, c), c) and np.array_equal(buf.down(ps, s), s)


@pytest.mark.parametrize("rows", [1, 33, 64])
def test_host_rows(dev, rows):
    rng = np.random.default_rng(rows)
    w = weights(rng, 70, 96)
    x = rng.normal(0, 1, (rows, 96)).astype(np.float32)
    wv, xd = mx.values(*w), x.astype(np.float64)
    assert (np.abs(matrix(dev, w).gemv(x) - xd @ wv.T) <= mx.product_bound(xd, wv)).all()


def hip(name, *args):
    """A HIP call in the runtime that the backend library is linked to (another copy may be loaded)."""
    from pagoda_amd import lib

    assert getattr(lib(), name)(*args) == 0, name


class Graph:
    """What `calls` queues on the handle's stream, captured."""

    def __init__(self, dev, calls):
        self.stream = C.c_void_p(dev.stream)
        self.exec = C.c_void_p()
        graph = C.c_void_p()
        dev.sync()
        hip("hipStreamBeginCapture", self.stream, 1)  # (thread-local mode)
        try:
            calls()
        finally:
            hip("hipStreamEndCapture", self.stream, C.byref(graph))
        hip("hipGraphInstantiate", C.byref(self.exec), graph, None, None, C.c_size_t(0))
        hip("hipGraphDestroy", graph)

    def replay(self):
        hip("hipGraphLaunch", self.exec, self.stream)

    def close(self):
        hip("hipGraphExecDestroy", self.exec)


def test_captured_calls_replay(dev, buf):
    """Two graphs of calls that need no scratch memory, replayed in turn with eager products of
    more rows (whose scratch may move) between: every replay of new rows is right, and an
    unchanged input gives the same bits."""
    from pagoda_amd import Matrix
    from pagoda_amd.matrix import mxfp4_quantize_dev

    rng = np.random.default_rng(4)
    h, i, rows = 256, 4096, 70
    planes = [mx.quantize(rng.normal(0, 0.05, s).astype(np.float32)) for s in ((i, h), (i, h), (h, i))]
    gate, up, down = (matrix(dev, p) for p in planes)
    gv, uv, dv = (mx.values(*p) for p in planes)
    zeros = lambda *s: np.zeros(s, np.float32)
    px, pmid, py, pb, ps4 = buf.up(zeros(rows, h)), buf.up(zeros(rows, i)), buf.up(zeros(rows, h)), buf.up(zeros(rows, h)), buf.up(zeros(4, i))
    pc, ps = buf.up(np.zeros((rows, i // 2), np.uint8)), buf.up(np.zeros((rows, i // 32), np.uint8))
    mid_bf = buf.up(np.zeros((rows, i), np.uint16))

    def block():
        mxfp4_quantize_dev(dev, px, F32, h, rows, h, pc, i // 2, ps, i // 32)
        Matrix.gemv_swiglu_mx_dev(gate, up, pc, i // 2, ps, i // 32, rows, pmid, i)
        mxfp4_quantize_dev(dev, pmid, F32, i, rows, i, pc, i // 2, ps, i // 32)
        down.gemv_mx_dev(pc, i // 2, ps, i // 32, rows, py, h)

    def rest():
        down.gemv_dev(mid_bf, i, rows, pb, h, BF16)
        Matrix.gemv_swiglu_dev(gate, up, px, h, 4, ps4, i)

    graphs = [Graph(dev, block), Graph(dev, rest)]
    before = None
    for step in range(4):
        if step != 2:
            x = rng.normal(0, 1, (rows, h)).astype(np.float32)
            bf = mx.bf16(rng.normal(0, 1, (rows, i)).astype(np.float32))
            for p, a in ((px, x), (mid_bf, bf)):
                put(dev, p, a)
        for g in graphs:
            g.replay()
        big = rng.normal(0, 1, (100 * (step + 1), i)).astype(np.float32)
        bd = big.astype(np.float64)
        assert (np.abs(run_rows(dev, buf, down, big, F32) - bd @ dv.T) <= mx.product_bound(bd, dv)).all()
        mid, y, b, s4 = (buf.down(p, zeros(r, c)) for p, r, c in ((pmid, rows, i), (py, rows, h), (pb, rows, h), (ps4, 4, i)))
        if step == 2:
            for now, then in zip((mid, y, b, s4), before):
                assert np.array_equal(now, then)
        before = mid, y, b, s4
        xv = mx.values(*mx.quantize(x))
        assert (np.abs(mid - mx.silu(xv @ gv.T) * (xv @ uv.T)) <= mx.swiglu_bound(xv, gv, uv)).all()
        mv = mx.values(*mx.quantize(mid))
        assert (np.abs(y - mv @ dv.T) <= mx.product_bound(mv, dv)).all()
        bv = mx.bf16_f32(bf).astype(np.float64)
        assert (np.abs(b - bv @ dv.T) <= mx.product_bound(bv, dv)).all()
        x4 = x[:4].astype(np.float64)
        assert (np.abs(s4 - mx.silu(x4 @ gv.T) * (x4 @ uv.T)) <= mx.swiglu_bound(x4, gv, uv)).all()
    for g in graphs:
        g.close()


def test_capture_refuses_rows_that_need_scratch(dev, buf):
    """Refused before anything is queued: the capture goes on, and the call works after it."""
    from pagoda_amd import PagodaError

    rng = np.random.default_rng(6)
    w = weights(rng, 48, 96)
    m, wv = matrix(dev, w), mx.values(*w)
    x = rng.normal(0, 1, (40, 96)).astype(np.float32)
    px, py = buf.up(x), buf.up(np.zeros((40, 48), np.float32))
    seen = []

    def calls():
        for t, rows in ((F32, 6), (F16, 9), (BF16, 5)):
            with pytest.raises(PagodaError) as e:
                m.gemv_dev(px, 96, rows, py, 48, t)
            seen.append(e.value.code)
        m.gemv_dev(px, 96, 5, py, 48, F32)

    g = Graph(dev, calls)
    assert len(set(seen)) == 1 and len(seen) == 3
    for _ in range(3):
        g.replay()
    got, xd = buf.down(py, np.zeros((40, 48), np.float32)), x.astype(np.float64)
    assert (np.abs(got[:5] - xd[:5] @ wv.T) <= mx.product_bound(xd[:5], wv)).all() and not got[5:].any()
    g.close()
    assert (np.abs(run_rows(dev, buf, m, x, F32) - xd @ wv.T) <= mx.product_bound(xd, wv)).all()


@pytest.mark.parametrize("handles", [1, 2])
def test_threads_at_once(dev, handles):
    """Products that share the stream's scratch (one handle) or have their own (two), queued
    by four threads: the bits of the same calls made alone."""
    from pagoda_amd import Device, Matrix

    devs = [Device("hip") for _ in range(handles)]
    rng = np.random.default_rng(8)
    w = weights(rng, 200, 4096)
    jobs = []
    for i, (t, rows) in enumerate(((F32, 333), (F16, 200), (F32, 17), (PLANES, 333))):
        d = devs[i % handles]
        raw, _ = rows_and_values(rng, t, rows, 4096)
        b = Buffers(d)
        jobs.append((d, b, Matrix.upload_mxfp4(d, *w, 200, 4096), t, raw))
    alone = [product(d, b, m, t, raw) for d, b, m, t, raw in jobs]
    bad = []

    def run(i):
        d, b, m, t, raw = jobs[i]
        try:
            for _ in range(20):
                if not np.array_equal(product(d, b, m, t, raw), alone[i]):
                    bad.append(i)
        except Exception as e:  # (a thread's exception would be lost)
            bad.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for _, b, m, _, _ in jobs:
        b.close()
        m.free()
    for d in devs:
        d.close()
    assert not bad


# ---- sizes whose offsets pass 32 bits, most of them zeros: sums of few products, checked in full precision


@pytest.fixture
def big():
    """A handle of its own, so that its scratch goes with it."""
    from pagoda_amd import Device

    d = Device("hip")
    yield d, Buffers(d)
    d.sync()


def fill(dev, ptr, byte, nbytes):
    hip("hipMemsetAsync", C.c_void_p(ptr), byte, C.c_size_t(nbytes), C.c_void_p(dev.stream))


def put(dev, ptr, a):
    from pagoda_amd._lib import call

    a = np.ascontiguousarray(a)
    call("pgd_device_memcpy", dev.handle, C.c_void_p(ptr), a.ctypes.data_as(C.c_void_p), C.c_size_t(a.nbytes), 0)


@pytest.mark.parametrize("t", [F32, F16, BF16, PLANES])
def test_rows_past_32_bits(big, t):
    """Rows at the ends and on both sides of the element (byte, for planes) 2^32."""
    dev, buf = big
    rng = np.random.default_rng(t)
    n, k = 48, 8192
    size = {F32: 4, F16: 2, BF16: 2, PLANES: 0.5}[t]
    mid = (2 ** 31 if t != PLANES else 2 ** 32) // (k if t != PLANES else k // 2)
    mid = mid // 2 if t == F32 else mid  # (f32: byte 2^32; its digits' too)
    rows = mid + 77
    w = weights(rng, n, k)
    m = matrix(dev, w)
    px, py = dev.alloc(int(rows * k * size)), dev.alloc(rows * n * 4)
    buf.ptrs += [px, py]
    fill(dev, px, 0, int(rows * k * size))
    checks = [(0, 40), (mid - 20, 40), (rows - 30, 30)]
    if t == PLANES:
        psc = dev.alloc(rows * (k // 32))
        buf.ptrs.append(psc)
        fill(dev, psc, 127, rows * (k // 32))
    wv, xs = mx.values(*w), []
    for r0, r in checks:
        raw, x = rows_and_values(rng, t, r, k)
        xs.append(x)
        put(dev, px + int(r0 * k * size), raw[0] if t == PLANES else raw)
        if t == PLANES:
            put(dev, psc + r0 * (k // 32), raw[1])
    if t == PLANES:
        m.gemv_mx_dev(px, k // 2, psc, k // 32, rows, py, n)
    else:
        m.gemv_dev(px, k, rows, py, n, t)
    for (r0, r), x in zip(checks, xs):
        got = dev.download(py + r0 * n * 4, (r, n), np.float32)
        assert (np.abs(got - x @ wv.T) <= mx.product_bound(x, wv)).all()
    assert not dev.download(py + 40 * n * 4, (1000, n), np.float32).any()
    buf.close()


def test_quantize_past_32_bits(big):
    from pagoda_amd.matrix import mxfp4_quantize_dev

    dev, buf = big
    rng = np.random.default_rng(11)
    k = 8192
    rows = 2 ** 31 // k + 33  # f32 elements past 2^31, bytes past 2^33
    px, pv, pc, ps = dev.alloc(rows * k * 4), dev.alloc(rows * k * 4), dev.alloc(rows * k // 2), dev.alloc(rows * k // 32)
    buf.ptrs += [px, pv, pc, ps]
    fill(dev, px, 0, rows * k * 4)
    xs = []
    for r0 in (0, rows // 2, rows - 33):
        xs.append((r0, rng.normal(0, 1, (33, k)).astype(np.float32)))
        put(dev, px + r0 * k * 4, xs[-1][1])
    mxfp4_quantize_dev(dev, px, F32, k, rows, k, pc, k // 2, ps, k // 32, pv, k)
    for r0, x in xs:
        c, s = mx.quantize(x)
        assert np.array_equal(dev.download(pc + r0 * (k // 2), c.shape, np.uint8), c)
        assert np.array_equal(dev.download(ps + r0 * (k // 32), s.shape, np.uint8), s)
        assert np.array_equal(dev.download(pv + r0 * k * 4, x.shape, np.float32), mx.values(c, s).astype(np.float32))
    buf.close()


@pytest.mark.parametrize("rows", [3, 100])
def test_matrix_past_32_bits(big, rows):
    from pagoda_amd import Matrix

    dev, buf = big
    rng = np.random.default_rng(rows)
    k = 8192
    n = 2 ** 32 // (k // 2) + 41
    pc, ps = dev.alloc(n * (k // 2)), dev.alloc(n * (k // 32))
    buf.ptrs += [pc, ps]
    fill(dev, pc, 0, n * (k // 2))
    fill(dev, ps, 127, n * (k // 32))
    ws = []
    for r0 in (0, n - 60, n // 2):
        ws.append((r0, weights(rng, 60, k)))
        put(dev, pc + r0 * (k // 2), ws[-1][1][0])
        put(dev, ps + r0 * (k // 32), ws[-1][1][1])
    m = Matrix.from_mxfp4_dev(dev, pc, k // 2, ps, k // 32, n, k)
    assert np.array_equal(m.dequant(n - 60, 60), mx.values(*ws[1][1]).astype(np.float32))
    for t in (F32, PLANES):
        raw, x = rows_and_values(rng, t, rows, k)
        py = dev.alloc(rows * n * 4)
        buf.ptrs.append(py)
        if t == PLANES:
            m.gemv_mx_dev(buf.up(raw[0]), k // 2, buf.up(raw[1]), k // 32, rows, py, n)
        else:
            m.gemv_dev(buf.up(raw), k, rows, py, n, t)
        for r in (0, rows - 1):
            got = dev.download(py + r * n * 4, (n,), np.float32)
            live = np.zeros(n, bool)
            for r0, p in ws:
                wv = mx.values(*p)
                assert (np.abs(got[r0:r0 + 60] - (x[r:r + 1] @ wv.T)[0]) <= mx.product_bound(x[r:r + 1], wv)[0]).all()
                live[r0:r0 + 60] = True
            assert not got[~live].any()
    m.free()
    buf.close()


@pytest.mark.parametrize("t,rows,k", [(F32, 17, 2 ** 24 + 160), (BF16, 40, 2 ** 23 + 128), (PLANES, 70, 2 ** 26 + 128)])
def test_rows_too_long_for_32_bit_lanes(big, t, rows, k):
    """Strides that a lane's 32-bit offsets of the many-row kernel cannot hold: 300 nonzeros
    a row, so the sums have few roundings (sums of zeros are exact)."""
    from pagoda_amd import Matrix

    dev, buf = big
    rng = np.random.default_rng(k)
    n, live = 20, 300
    cols = np.sort(np.concatenate([rng.choice(k - 64, live - 64, replace=False), np.arange(k - 64, k)]))
    nblk = k // 32
    codes, scales = rng.integers(0, 256, (n, k // 2), dtype=np.uint8), np.full((n, nblk), 124, np.uint8)
    m = Matrix.upload_mxfp4(dev, codes, scales, n, k)
    nib = lambda c, j: (c[:, j // 2] >> (4 * (j % 2)).astype(np.uint8)) & 15
    wv = mx.E2M1[nib(codes, cols)] / 8
    py = buf.up(np.zeros((rows, n), np.float32))
    if t == PLANES:
        ldc, lds = pad16(k // 2), pad16(nblk)
        pc, ps = dev.alloc(rows * ldc), dev.alloc(rows * lds)
        buf.ptrs += [pc, ps]
        fill(dev, pc, 0, rows * ldc)
        fill(dev, ps, 127, rows * lds)
        x = np.zeros((rows, live))
        for r in range(rows):
            row = np.zeros(ldc, np.uint8)
            c = rng.integers(0, 16, live).astype(np.uint8)
            np.bitwise_or.at(row, cols // 2, c << (4 * (cols % 2)).astype(np.uint8))
            x[r] = mx.E2M1[c]
            put(dev, pc + r * ldc, row)
        m.gemv_mx_dev(pc, ldc, ps, lds, rows, py, n)
    else:
        raw, xf = mx.rows_of(rng.normal(0, 1, (rows, live)).astype(np.float32), t)
        x = xf.astype(np.float64)
        size = raw.dtype.itemsize
        px = dev.alloc(rows * k * size)
        buf.ptrs.append(px)
        for r in range(rows):
            row = np.zeros(k, raw.dtype)
            row[cols] = raw[r]
            put(dev, px + r * k * size, row)
        m.gemv_dev(px, k, rows, py, n, t)
    got = buf.down(py, np.zeros((rows, n), np.float32))
    # (a product of f32 rows is up to 3 terms' products; 8 waves' or ranges' sums are joined)
    bound = (3 * live + 32) * 2.0 ** -23 * (np.abs(x) @ np.abs(wv).T)
    assert (np.abs(got - x @ wv.T) <= bound).all()
    m.free()
    buf.close()
