"""MXFP4 operators on the GPU against their definitions in float64 (mxfp4.py):
quantization bit for bit, products within the bound of f32 sums."""
import ctypes as C

import numpy as np
import pytest

import mxfp4 as mx

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 2


class Buffers:
    """Device buffers of one test, freed at its end."""

    def __init__(self, dev):
        self.dev, self.ptrs = dev, []

    def up(self, a):
        self.ptrs.append(self.dev.upload(a))
        return self.ptrs[-1]

    def down(self, p, a):
        return self.dev.download(p, a.shape, a.dtype)

    def close(self):
        self.dev.sync()
        for p in self.ptrs:
            self.dev.free(p)


@pytest.fixture
def buf(dev):
    b = Buffers(dev)
    yield b
    b.close()


def pad16(n):
    return (n + 15) // 16 * 16


def weights(rng, n, k, spread=3):
    """Planes of random codes, with scales 2^-spread .. 2^spread around 2^-6."""
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    scales = rng.integers(121 - spread, 122 + spread, (n, k // 32)).astype(np.uint8)
    return codes, scales


def matrix(dev, planes):
    from pagoda_amd import Matrix

    codes, scales = planes
    return Matrix.upload_mxfp4(dev, codes, scales, codes.shape[0], codes.shape[1] * 2)


def special_rows(rng, rows, k):
    """Rows of ordinary values over many binades, with blocks of zeros, ties,
    subnormals and the largest numbers among them."""
    x = (rng.normal(0, 1, (rows, k)) * 2.0 ** rng.integers(-20, 20, (rows, k // 32)).repeat(32, 1)).astype(np.float32)
    b = x.reshape(-1, 32)
    n = b.shape[0]
    pick = lambda i: b[(i * 7 + 3) % n]
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7] * 4, np.float32)
    b[n // 2] = ties * np.where(np.arange(32) % 3, 1, -1) * 2.0 ** 5
    if n > 8:
        pick(1)[:] = 0
        pick(2)[:] = -0.0
        pick(3)[:] = ties * np.float32(2.0 ** -127)
        pick(4)[:] = rng.integers(0, 1 << 20, 32).astype(np.uint32).view(np.float32)
        pick(5)[:] = np.finfo(np.float32).max * np.linspace(-1, 1, 32, dtype=np.float32)
        pick(6)[:] = ties * np.float32(2.0 ** -120)
    return x


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 64), (1, 896), (70, 96), (5, 2080), (2, 4864), (300, 160), (0, 64)])
def test_quantize_bit_for_bit(dev, buf, t, rows, k):
    from pagoda_amd.matrix import mxfp4_quantize_dev

    rng = np.random.default_rng(rows * 1000 + k + t)
    x = special_rows(rng, max(rows, 1), k)
    top = {F32: np.finfo(np.float32).max, F16: 60000, BF16: mx.bf16_f32(np.uint16([0x7F7F]))[0]}[t]
    raw, x = mx.rows_of(np.clip(x, -np.float32(top), np.float32(top)), t)
    assert np.isfinite(x).all()
    ldx, ldc, lds, ldv = k + 8, pad16(k // 2) + 16, pad16(k // 32) + 16, k + 4
    dx = buf.up(mx.padded(raw, ldx, raw.dtype.type(77)))
    shape = (max(rows, 1),)
    codes, scales = np.full(shape + (ldc,), 0xA5, np.uint8), np.full(shape + (lds,), 0x5A, np.uint8)
    vals = np.full(shape + (ldv,), 123.0, np.float32)
    dc, ds, dv = buf.up(codes), buf.up(scales), buf.up(vals)
    want_c, want_s = mx.quantize(np.ascontiguousarray(x))
    want_v = mx.values(want_c, want_s).astype(np.float32)
    mxfp4_quantize_dev(dev, dx, t, ldx, rows, k, dc, ldc, ds, lds, dv, ldv)
    gc, gs, gv = buf.down(dc, codes), buf.down(ds, scales), buf.down(dv, vals)
    codes[:rows, :k // 2], scales[:rows, :k // 32], vals[:rows, :k] = want_c[:rows], want_s[:rows], want_v[:rows]
    assert np.array_equal(gs, scales)  # bytes past the rows left as they were
    assert np.array_equal(gc, codes)
    assert np.array_equal(gv, vals)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_quantize_nonfinite_blocks(dev, buf, t):
    """An infinity or NaN makes its block NaN and no other."""
    from pagoda_amd.matrix import mxfp4_quantize_dev

    rng = np.random.default_rng(5)
    x = rng.normal(0, 1, (4, 128)).astype(np.float32)
    raw, v = mx.rows_of(x, t)
    raw = raw.copy()
    bad = {F32: [np.inf, np.nan], F16: [np.inf, np.nan], BF16: [0x7F80, 0x7FC1]}[t]
    raw[0, 5], raw[2, 127] = bad
    raw[3, 64] = {F32: -np.inf, F16: -np.inf, BF16: 0xFF80}[t]
    hit = [(0, 0), (2, 3), (3, 2)]
    codes, scales = np.zeros((4, 64), np.uint8), np.zeros((4, 16), np.uint8)
    dx, dc, ds, dv = buf.up(raw), buf.up(codes), buf.up(scales), buf.up(x)
    mxfp4_quantize_dev(dev, dx, t, 128, 4, 128, dc, 64, ds, 16, dv, 128)
    gc, gs, gv = buf.down(dc, codes), buf.down(ds, scales), buf.down(dv, x)
    want_c, s = mx.quantize(v)
    want_s = mx.padded(s, 16, np.uint8(0))
    for r, b in hit:
        want_s[r, b] = 255
        want_c[r, 16 * b:16 * b + 16] = 0
    assert np.array_equal(gs, want_s) and np.array_equal(gc, want_c)
    nan = np.isnan(gv).reshape(4, 4, 32)
    assert all(nan[r, b].all() for r, b in hit) and nan.sum() == 32 * len(hit)


@pytest.mark.parametrize("n,k", [(1, 32), (16, 128), (33, 160), (100, 896), (7, 2080)])
def test_matrix_holds_its_planes(dev, buf, n, k):
    """Dequantized rows equal the definition for every scale byte, from host and device planes."""
    from pagoda_amd import Matrix

    rng = np.random.default_rng(n + k)
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    scales = rng.permutation(np.resize(np.arange(255, dtype=np.uint8), n * (k // 32))).reshape(n, k // 32)
    if n > 1:
        scales[1, 0] = 255
    with np.errstate(over="ignore"):
        want = mx.values(codes, scales).astype(np.float32)
    m = Matrix.upload_mxfp4(dev, codes, scales, n, k)
    assert (m.fmt, m.n_out, m.n_in) == (5, n, k) and m.algo_bytes == n * k * 4.25 / 8
    ldc, lds = pad16(k // 2) + 32, pad16(k // 32) + 16
    d = Matrix.from_mxfp4_dev(dev, buf.up(mx.padded(codes, ldc, np.uint8(0xFF))), ldc,
                              buf.up(mx.padded(scales, lds, np.uint8(0xFF))), lds, n, k)
    for w in (m, d):
        assert np.array_equal(w.dequant(), want, equal_nan=True)
        if n > 3:
            assert np.array_equal(w.dequant(2, n - 3), want[2:n - 1], equal_nan=True)


def run_rows(dev, buf, m, raw, t, res=None, up=None, ldx_more=0, ldy_more=0, in_place=False, y_off=0):
    """gemv_dev / gemv_swiglu_dev over strided rows whose gaps are NaN; the output's gap must stay."""
    from pagoda_amd import Matrix

    rows, n, k = raw.shape[0], m.n_out, m.n_in
    ldx, ldy = (k + 7) // 8 * 8 + ldx_more, n + ldy_more
    nan = raw.dtype.type(0x7FC0) if t == BF16 else raw.dtype.type(np.nan)
    y = np.full((rows + 1, ldy), 55.0, np.float32)
    if in_place:
        y[:rows, :n] = res
    py = buf.up(np.concatenate([np.zeros(y_off, np.float32), y.ravel()])) + 4 * y_off
    px = buf.up(mx.padded(raw, ldx, nan))
    pr = py if in_place else buf.up(mx.padded(res, ldy, np.float32(9))) if res is not None else 0
    if up is not None:
        Matrix.gemv_swiglu_dev(m, up, px, ldx, rows, py, ldy)
    else:
        m.gemv_dev(px, ldx, rows, py, ldy, t, pr, ldy)
    got = buf.down(py, y)
    assert (got[rows:] == 55.0).all() and (got[:, n:] == 55.0).all()
    return got[:rows, :n]


def run_planes(dev, buf, m, planes, res=None, up=None, ldc_more=0, ldy_more=0, y_off=0):
    from pagoda_amd import Matrix

    codes, scales = planes
    rows, n, k = codes.shape[0], m.n_out, m.n_in
    ldc, lds, ldy = k // 2 + ldc_more, pad16(k // 32), n + ldy_more
    y = np.full((rows + 1, ldy), 55.0, np.float32)
    py = buf.up(np.concatenate([np.zeros(y_off, np.float32), y.ravel()])) + 4 * y_off
    pc, ps = buf.up(mx.padded(codes, ldc, np.uint8(0x77))), buf.up(mx.padded(scales, lds, np.uint8(0xFF)))
    pr = buf.up(mx.padded(res, ldy, np.float32(9))) if res is not None else 0
    if up is not None:
        Matrix.gemv_swiglu_mx_dev(m, up, pc, ldc, ps, lds, rows, py, ldy)
    else:
        m.gemv_mx_dev(pc, ldc, ps, lds, rows, py, ldy, pr, ldy)
    got = buf.down(py, y)
    assert (got[rows:] == 55.0).all() and (got[:, n:] == 55.0).all()
    return got[:rows, :n]


# rows on both sides of every row tile and launch limit; widths inside and at the end of a k tile
ROWS = [1, 2, 5, 6, 16, 17, 21, 22, 32, 33, 64, 65, 130, 200]
SHAPES = [(1, 32), (40, 96), (100, 896), (257, 416), (333, 1024)]


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("n,k", SHAPES)
def test_gemv_rows(dev, buf, t, rows, n, k):
    rng = np.random.default_rng(rows * 7 + n + k + t)
    w = weights(rng, n, k)
    raw, x = mx.rows_of(rng.normal(0, 1, (rows, k)).astype(np.float32), t)
    m, wv, x = matrix(dev, w), mx.values(*w), x.astype(np.float64)
    bound = mx.product_bound(x, wv)
    got = run_rows(dev, buf, m, raw, t, ldx_more=8 * (rows % 3), ldy_more=rows % 2)
    assert (np.abs(got - x @ wv.T) <= bound).all()
    res = rng.normal(0, 1, (rows, n)).astype(np.float32)
    got = run_rows(dev, buf, m, raw, t, res=res, ldy_more=3, in_place=bool(rows % 2), y_off=rows % 4)
    assert (np.abs(got - (res + x @ wv.T)) <= bound + 2.0 ** -23 * np.abs(res + x @ wv.T)).all()


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("n,k", SHAPES)
def test_gemv_planes(dev, buf, rows, n, k):
    rng = np.random.default_rng(rows * 5 + n + k)
    w, x = weights(rng, n, k), weights(rng, rows, k, spread=5)
    m, wv, xv = matrix(dev, w), mx.values(*w), mx.values(*x)
    bound = mx.product_bound(xv, wv)
    got = run_planes(dev, buf, m, x, ldc_more=16 * (rows % 3), ldy_more=rows % 2)
    assert (np.abs(got - xv @ wv.T) <= bound).all()
    res = rng.normal(0, 1, (rows, n)).astype(np.float32)
    got = run_planes(dev, buf, m, x, res=res, ldy_more=3, y_off=rows % 4)
    assert (np.abs(got - (res + xv @ wv.T)) <= bound + 2.0 ** -23 * np.abs(res + xv @ wv.T)).all()


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("n,k", [(1, 32), (100, 896), (257, 416)])
def test_gate_up_pair(dev, buf, rows, n, k):
    rng = np.random.default_rng(rows * 3 + n + k)
    g, u = weights(rng, n, k), weights(rng, n, k)
    gm, um, gv, uv = matrix(dev, g), matrix(dev, u), mx.values(*g), mx.values(*u)
    x = rng.normal(0, 1, (rows, k)).astype(np.float32)
    xd = x.astype(np.float64)
    want = mx.silu(xd @ gv.T) * (xd @ uv.T)
    got = run_rows(dev, buf, gm, x, F32, up=um, ldx_more=8, ldy_more=rows % 2)
    assert (np.abs(got - want) <= mx.swiglu_bound(xd, gv, uv)).all()
    p = weights(rng, rows, k, spread=5)
    xd = mx.values(*p)
    want = mx.silu(xd @ gv.T) * (xd @ uv.T)
    got = run_planes(dev, buf, gm, p, up=um, ldc_more=16, ldy_more=rows % 2)
    assert (np.abs(got - want) <= mx.swiglu_bound(xd, gv, uv)).all()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_rows_enter_exactly(dev, buf, t, rows):
    """One nonzero per row: outputs are x w within the roundings of adding its terms'
    products (at most 4 of 2^-23), so no bit of x is lost, over x's whole range of
    exponents; tiny values keep their relative accuracy down to bf16's own range."""
    rng = np.random.default_rng(rows + t)
    n, k = 80, 256
    w = weights(rng, n, k, spread=1)
    e = rng.integers(-100, 100, rows) if t != F16 else rng.integers(-14, 15, rows)
    v = (rng.uniform(1, 2, rows) * np.where(rng.random(rows) < 0.5, -1, 1) * 2.0 ** e).astype(np.float32)
    x = np.zeros((rows, k), np.float32)
    x[np.arange(rows), rng.integers(0, k, rows)] = v
    raw, x = mx.rows_of(x, t)
    want = x.astype(np.float64) @ mx.values(*w).T
    got = run_rows(dev, buf, matrix(dev, w), raw, t)
    assert (np.abs(got - want) <= 4 * 2.0 ** -23 * np.abs(want)).all()


@pytest.mark.parametrize("rows", [1, 30, 200])
def test_nonfinite_stays_in_its_row_and_column(dev, buf, rows):
    """A NaN or infinity among a row's values makes that row's outputs non-finite (NaN for a
    NaN; an infinity keeps its sign in f16, bf16 and few f32 rows, and may be a NaN in many f32
    rows), a NaN block of weights its output's; no other row or output."""
    rng = np.random.default_rng(rows)
    n, k = 100, 160
    codes, scales = weights(rng, n, k)
    codes[:, 80 // 2] = 0x22  # the infinity's weights are 1
    scales[17, 3] = 255
    m, wv = matrix(dev, (codes, scales)), mx.values(codes, scales)
    x = rng.normal(0, 1, (rows, k)).astype(np.float32)
    x[0, 80] = np.inf
    if rows > 1:
        x[rows - 1, 159] = np.nan
    for t in (F32, F16, BF16):
        raw, xv = mx.rows_of(np.nan_to_num(x, nan=0, posinf=0), t)
        raw = raw.copy()
        raw[0, 80] = np.inf if t != BF16 else 0x7F80
        if rows > 1:
            raw[rows - 1, 159] = np.nan if t != BF16 else 0x7FC0
        got = run_rows(dev, buf, m, raw, t)
        live = [c for c in range(n) if c != 17]
        assert np.isnan(got[:, 17]).all()
        assert (got[0, live] == np.inf).all() or (t == F32 and rows > 16 and np.isnan(got[0, live]).all())
        if rows > 1:
            assert np.isnan(got[rows - 1]).all()
        mid = slice(1, rows - 1)
        assert np.isfinite(got[mid][:, live]).all()
    p = mx.quantize(np.ascontiguousarray(np.clip(np.nan_to_num(x, nan=0), -9, 9), np.float32))
    p[1][0, 2] = 255
    got = run_planes(dev, buf, m, p)
    assert np.isnan(got[0]).all() and np.isnan(got[:, 17]).all()
    assert np.isfinite(got[1:][:, live]).all()


def test_extreme_scales(dev, buf):
    """Scale bytes near both ends on one side, undone by the other side's: sums in range."""
    rng = np.random.default_rng(9)
    for lo, hi in ((2, 250), (250, 2)):
        w = rng.integers(0, 256, (40, 64), dtype=np.uint8), np.full((40, 4), lo, np.uint8)
        x = rng.integers(0, 256, (9, 64), dtype=np.uint8), np.full((9, 4), hi, np.uint8)
        wv, xv = mx.values(*w), mx.values(*x)
        got = run_planes(dev, buf, matrix(dev, w), x)
        assert (np.abs(got - xv @ wv.T) <= mx.product_bound(xv, wv)).all()


def test_feed_forward_in_mxfp4(dev, buf):
    """The operators together as a feed-forward block: rows quantized, gate/up pair, its rows
    quantized, down projection plus residual; every step against float64 on the step's own input."""
    from pagoda_amd import Matrix
    from pagoda_amd.matrix import mxfp4_quantize_dev

    rng = np.random.default_rng(3)
    for rows in (1, 37, 150):
        h, i = 256, 416
        x = rng.normal(0, 1, (rows, h)).astype(np.float32)
        planes = [mx.quantize(rng.normal(0, 0.05, s).astype(np.float32)) for s in ((i, h), (i, h), (h, i))]
        gate, up, down = (matrix(dev, p) for p in planes)
        gv, uv, dv = (mx.values(*p) for p in planes)
        px, pmid, py = buf.up(x), buf.up(np.zeros((rows, i), np.float32)), buf.up(x)
        pc, ps = buf.up(np.zeros((rows, i), np.uint8)), buf.up(np.zeros((rows, 16), np.uint8))
        mxfp4_quantize_dev(dev, px, F32, h, rows, h, pc, h // 2, ps, 16)
        Matrix.gemv_swiglu_mx_dev(gate, up, pc, h // 2, ps, 16, rows, pmid, i)
        mxfp4_quantize_dev(dev, pmid, F32, i, rows, i, pc, i // 2, ps, 16)
        down.gemv_mx_dev(pc, i // 2, ps, 16, rows, py, h, py, h)
        mid, y = buf.down(pmid, np.zeros((rows, i), np.float32)), buf.down(py, x)
        xv = mx.values(*mx.quantize(x))
        assert (np.abs(mid - mx.silu(xv @ gv.T) * (xv @ uv.T)) <= mx.swiglu_bound(xv, gv, uv)).all()
        mv = mx.values(*mx.quantize(mid))
        want = x + mv @ dv.T
        assert (np.abs(y - want) <= mx.product_bound(mv, dv) + 2.0 ** -23 * np.abs(want)).all()
