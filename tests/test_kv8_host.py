"""The 8-bit KV cache without a GPU: the definition the GPU tests compare with, refusals before the first HIP
call, and addresses of the Python layer."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest

import kv8

ARG, SHAPE = -1, -4
A = 1 << 20  # a device address that is never followed


def test_rounding_to_codes():
    codes = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    codes = np.array(codes[:127])  # (the last stands for NaN)
    assert codes.max() == 448
    assert np.array_equal(kv8.round_e4m3(codes), codes)
    mid = (codes[1:] + codes[:-1]) / 2
    assert np.array_equal(kv8.round_e4m3(mid), np.where(np.arange(126) % 2 == 0, codes[:-1], codes[1:]))
    near = np.nextafter(mid, 0)
    assert np.array_equal(kv8.round_e4m3(-near), -codes[:-1])


@pytest.mark.parametrize("most", [448.0, 127.0])
def test_smallest_power_of_two(most):
    for e in (-126, -60, -1, 0, 7, 119):
        top = most * 2.0 ** e
        assert kv8.holds(top, most) == e
        assert kv8.holds(np.nextafter(top, np.inf), most) == e + 1
        assert kv8.holds(np.nextafter(top, 0), most) == e
    assert kv8.holds(0.0, most) == kv8.holds(2.0 ** -149, most) == -126
    assert kv8.holds(float(np.finfo(np.float32).max), 448.0) == 120


def test_page_grows_and_starts_anew():
    c = kv8.Cache(2, 1, 64)
    one, big = np.ones((1, 64)), np.full((1, 64), 1000.0)
    c.append(one, one, [16])
    assert c.exps[0, 1, 0] == -8 and np.array_equal(c.read(0, [16]), one)
    c.append(big, one, [17])
    assert c.exps[0, 1, 0] == 2 and c.exps[1, 1, 0] == -8
    assert np.array_equal(c.read(0, [16, 17]), np.concatenate([one, np.full((1, 64), 1024.0)]))
    c.append(one, one, [16])
    assert c.exps[0, 1, 0] == -8 and not c.units[0, 1, 0, 1].any()


# ---- refusals -----------------------------------------------------------------------


def lib():
    from pagoda_amd import _lib

    return _lib.lib()


@pytest.fixture
def dev():
    """A handle whose fields no refused call reads."""
    return C.cast(C.create_string_buffer(4096), C.c_void_p)


APPEND = dict(pool=A, n_pages=4, kv_heads=2, head_dim=64, k=A, ldk=128, v=A, ldv=128, type=0, slots=A, rows=3)
READ = dict(pool=A, n_pages=4, kv_heads=2, head_dim=64, slots=A, rows=3, k=A, ldk=128, v=A, ldv=128)
ATTN = dict(pool=A, n_pages=4, kv_heads=2, head_dim=64, heads=4, q=A, ldq=256, type=0, nseq=2, row_start=A, lens=A,
            tables=A, max_blocks=40, rows=3, max_rows=2, out=A, ldo=256, gate=A, ldg=256, ws=A, ws_bytes=1 << 40)
SELECT = dict(pool=A, n_pages=4, kv_heads=2, head_dim=64, heads=4, q=A, ldq=256, type=0, nseq=2, row_start=A, lens=A,
              tables=A, max_blocks=40, rows=3, top=8, sinks=1, recent=2, sel=A, count=A, ws=A, ws_bytes=1 << 40)
SPARSE = dict(pool=A, n_pages=4, kv_heads=2, head_dim=64, heads=4, q=A, ldq=256, type=0, nseq=2, row_start=A, lens=A,
              tables=A, max_blocks=4000, rows=3, top=2000, sel=A, count=A, out=A, ldo=256, gate=A, ldg=256, ws=A,
              ws_bytes=1 << 40)
TABLES = dict(block=16, nseq=2, lens=A, counts=A, tables=A, max_blocks=8, free=A, n_free=4, taken=A, rows=3,
              new_lens=A, new_taken=A, row_start=A, seq=A, pos=A, slots=A, status=A)
CALLS = {"pgd_kv8_append_dev": APPEND, "pgd_kv8_read_dev": READ, "pgd_attn_kv8_dev": ATTN,
         "pgd_kv8_select_dev": SELECT, "pgd_attn_kv8_sparse_dev": SPARSE, "pgd_kv_tables_dev": TABLES}

POOL = [(dict(pool=0), ARG), (dict(pool=A + 8), ARG), (dict(n_pages=0), SHAPE), (dict(n_pages=1 << 27), SHAPE),
        (dict(kv_heads=0), SHAPE), (dict(kv_heads=2000), SHAPE), (dict(head_dim=80), SHAPE), (dict(head_dim=512), SHAPE),
        (dict(rows=-1), ARG)]
QUERY = [(dict(heads=3), SHAPE), (dict(heads=0), SHAPE), (dict(q=0), ARG), (dict(q=A + 4), ARG), (dict(ldq=255), SHAPE),
         (dict(ldq=260), SHAPE), (dict(type=3), ARG), (dict(type=-1), ARG), (dict(nseq=-1), ARG), (dict(row_start=0), ARG),
         (dict(lens=0), ARG), (dict(tables=0), ARG), (dict(max_blocks=0), SHAPE), (dict(max_blocks=(1 << 26) + 1), SHAPE),
         (dict(rows=1 << 24), SHAPE), (dict(nseq=(1 << 24) + 1), SHAPE), (dict(ws=0), ARG), (dict(ws=A + 8), ARG), (dict(ws_bytes=16), SHAPE)]
RESULT = [(dict(out=0), ARG), (dict(out=A + 8), ARG), (dict(ldo=248), SHAPE), (dict(ldo=258), SHAPE),
          (dict(gate=A + 8), ARG), (dict(ldg=248), SHAPE)]
LIST = [(dict(rows=1 << 21, max_blocks=1 << 12), SHAPE), (dict(top=0), SHAPE), (dict(top=(1 << 20) + 1), SHAPE), (dict(sel=0), ARG), (dict(count=0), ARG)]
REFUSED = (
    [("pgd_kv8_append_dev", c, e) for c, e in POOL + [
        (dict(k=0), ARG), (dict(v=0), ARG), (dict(k=A + 8), ARG), (dict(v=A + 2), ARG), (dict(ldk=127), SHAPE),
        (dict(ldk=120), SHAPE), (dict(ldv=132), SHAPE), (dict(type=3), ARG), (dict(slots=0), ARG),
        (dict(rows=1 << 23), SHAPE)]]
    + [("pgd_kv8_read_dev", c, e) for c, e in POOL + [
        (dict(k=0), ARG), (dict(v=A + 4), ARG), (dict(ldk=126), SHAPE), (dict(ldv=130), SHAPE), (dict(slots=0), ARG),
        (dict(rows=1 << 28), SHAPE)]]
    + [("pgd_attn_kv8_dev", c, e) for c, e in POOL + QUERY + RESULT + [(dict(max_rows=-1), ARG)]]
    + [("pgd_kv8_select_dev", c, e) for c, e in POOL + QUERY + LIST + [
        (dict(sinks=-1), ARG), (dict(recent=-1), ARG), (dict(sinks=6, recent=3), ARG),
        (dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), ARG)]]
    + [("pgd_attn_kv8_sparse_dev", c, e) for c, e in POOL + QUERY + RESULT + LIST]
    + [("pgd_kv_tables_dev", c, ARG) for c in [
        dict(block=0), dict(block=-16), dict(nseq=-1), dict(max_blocks=0), dict(n_free=-1), dict(rows=-1), dict(lens=0),
        dict(counts=0), dict(tables=0), dict(free=0), dict(taken=0), dict(new_lens=0), dict(new_taken=0),
        dict(row_start=0), dict(seq=0), dict(pos=0), dict(slots=0), dict(status=0)]]
    + [("pgd_kv_tables_dev", c, SHAPE) for c in [dict(rows=(1 << 30) + 1), dict(nseq=(1 << 24) + 1)]])


@pytest.mark.parametrize("name,change,code", REFUSED, ids=[f"{n}-{c}" for n, c, _ in REFUSED])
def test_refusals(dev, name, change, code):
    args = dict(CALLS[name], **change)
    assert getattr(lib(), name)(dev, *args.values()) == code
    from pagoda_amd import _lib

    assert _lib.last_error()


@pytest.mark.parametrize("name", sorted(CALLS))
def test_null_device(name):
    assert getattr(lib(), name)(None, *CALLS[name].values()) == ARG


@pytest.mark.parametrize("name", sorted(set(CALLS) - {"pgd_kv_tables_dev"}))
def test_no_rows_is_nothing(dev, name):
    """Without rows nothing is queued, whatever the rows' addresses."""
    args = dict(CALLS[name], rows=0)
    for key in ("k", "v", "q", "out", "gate", "slots", "sel", "count", "ws"):
        if key in args:
            args[key] = 0
    assert getattr(lib(), name)(dev, *args.values()) == 0
    if "nseq" in args:
        assert getattr(lib(), name)(dev, *dict(args, rows=3, nseq=0).values()) == 0


def test_sizes():
    l = lib()
    for kv, hd in ((1, 64), (2, 64), (4, 128), (4, 256), (3, 256), (1024, 64)):
        size = l.pgd_kv8_page_bytes(kv, hd)
        assert size % 256 == 0 and 0 <= size - kv * (34 * hd + 4) < 256
    for kv, hd in ((0, 64), (-1, 64), (2, 96), (1025, 64)):
        assert l.pgd_kv8_page_bytes(kv, hd) == 0
    assert l.pgd_attn_kv8_ws_bytes(4, 2, 64, 1, 1, 1) >= 0
    assert l.pgd_attn_kv8_ws_bytes(5, 2, 64, 1, 100, 1) == 0 == l.pgd_kv8_sparse_ws_bytes(4, 2, 96, 1, 100, 8)
    # (one score per row, KV head and page)
    assert l.pgd_kv8_sparse_ws_bytes(4, 2, 64, 3, 100, 8) >= 3 * 2 * 100 * 4


HOST = [b"rows", "rows", (C.c_char * 64)(), np.zeros(4), 4096.0, C.c_void_p(A)]


def pool_calls():
    from pagoda_amd.kv8 import Kv8Pool, kv_tables_dev

    d = SimpleNamespace(handle=None)
    p = Kv8Pool(d, 2, 64, 4, A)
    return [
        (lambda k, v, s: p.append_dev(k, 128, v, 128, 0, s, 3), 3),
        (lambda s, k, v: p.read_dev(s, 3, k, 128, v, 128), 3),
        (lambda q, r, l, t, o, w, g: p.attn_dev(4, q, 256, 0, 2, r, l, t, 40, 3, 2, o, 256, w, 1 << 30, g, 256), 7),
        (lambda q, r, l, t, s, c, w: p.select_dev(4, q, 256, 0, 2, r, l, t, 40, 3, 8, 1, 2, s, c, w, 1 << 30), 7),
        (lambda q, r, l, t, s, c, o, w, g: p.attn_sparse_dev(4, q, 256, 0, 2, r, l, t, 40, 3, 8, s, c, o, 256, w, 1 << 30,
                                                             g, 256), 9),
        (lambda *a: kv_tables_dev(d, 16, 2, a[0], a[1], a[2], 8, a[3], 4, a[4], 3, *a[5:]), 12),
    ]


@pytest.mark.parametrize("which", range(6))
def test_host_memory_is_no_device_address(which):
    from pagoda_amd import PagodaError

    call, count = pool_calls()[which]
    for good in (A, np.int64(A), None):
        with pytest.raises(PagodaError) as e:
            call(*[good] * count)
        assert e.value.code == ARG  # (no device)
    for i in range(count):
        for bad in HOST:
            args = [A] * count
            args[i] = bad.copy() if isinstance(bad, np.ndarray) else bad
            with pytest.raises((TypeError, ValueError)):
                call(*args)


def test_pools_of_no_pages():
    from pagoda_amd import Kv8Pool

    for kv, hd, n in ((2, 96, 4), (0, 64, 4), (2, 64, 0)):
        with pytest.raises(ValueError):
            Kv8Pool(SimpleNamespace(handle=None), kv, hd, n, A)
