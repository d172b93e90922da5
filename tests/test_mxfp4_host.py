"""MXFP4 entry points without a GPU: every refusal comes before the first HIP
call, and the NumPy definition the GPU tests use is checked against the format."""
import ctypes as C

import numpy as np
import pytest

import mxfp4 as mx

ARG, SHAPE, FORMAT = -1, -4, -7


class QMat(C.Structure):
    _fields_ = [("fmt", C.c_int), ("n_out", C.c_int), ("n_in", C.c_int), ("nsb", C.c_int), ("base", C.c_void_p),
                ("bytes", C.c_size_t), ("p", C.c_void_p * 4)]


class MatrixHandle(C.Structure):
    """A matrix handle's host side: what the argument checks read."""
    _fields_ = [("dev", C.c_void_p), ("m", QMat)]


def handle(fmt=5, n_out=48, n_in=64, dev=0x1000):
    return MatrixHandle(dev, QMat(fmt, n_out, n_in, 1, None, 0, (C.c_void_p * 4)()))


def code(name, *args):
    from pagoda_amd import _lib

    return getattr(_lib.lib(), name)(*args)


# never dereferenced: aligned and misaligned addresses
A = 0x10000


QUANT = dict(dev=A, x=A, t=0, ldx=64, rows=2, k=64, codes=A, ldc=32, scales=A, lds=16, values=None, ldv=0)


@pytest.mark.parametrize("change,want", [
    (dict(dev=None), ARG), (dict(x=None), ARG), (dict(codes=None), ARG), (dict(scales=None), ARG),
    (dict(t=3), ARG), (dict(t=-1), ARG), (dict(x=A + 4), ARG), (dict(codes=A + 8), ARG), (dict(scales=A + 8), ARG),
    (dict(values=A + 4, ldv=64), ARG), (dict(values=A, ldv=60), SHAPE), (dict(values=A, ldv=66), SHAPE),
    (dict(rows=-1), SHAPE), (dict(k=0), SHAPE), (dict(k=-32), SHAPE), (dict(k=48), SHAPE),
    (dict(ldx=56), SHAPE), (dict(ldx=68), SHAPE), (dict(ldc=16), SHAPE), (dict(ldc=40), SHAPE),
    (dict(lds=0), SHAPE), (dict(lds=4), SHAPE), (dict(lds=24), SHAPE),
])
def test_quantize_refuses(change, want):
    a = dict(QUANT, **change)
    assert code("pgd_mxfp4_quantize_dev", a["dev"], a["x"], a["t"], a["ldx"], a["rows"], a["k"], a["codes"], a["ldc"],
                a["scales"], a["lds"], a["values"], a["ldv"]) == want


PROD = dict(m={}, codes=A, ldc=32, scales=A, lds=16, rows=2, y=A, ldy=48, res=None, ldres=0)


@pytest.mark.parametrize("change,want", [
    (dict(m=None), ARG), (dict(y=None), ARG), (dict(codes=None), ARG), (dict(scales=None), ARG),
    (dict(m=dict(fmt=0)), FORMAT), (dict(m=dict(fmt=1)), FORMAT),
    (dict(codes=A + 4), ARG), (dict(scales=A + 4), ARG), (dict(ldc=24), SHAPE), (dict(ldc=16), SHAPE),
    (dict(lds=8), SHAPE), (dict(ldy=47), SHAPE), (dict(res=A, ldres=47), SHAPE),
])
def test_product_of_planes_refuses(change, want):
    a = dict(PROD, **change)
    m = handle(**a["m"]) if a["m"] is not None else None
    ptr = C.byref(m) if m is not None else None
    assert code("pgd_matrix_gemv_mx_dev", ptr, a["codes"], a["ldc"], a["scales"], a["lds"], a["rows"], a["y"],
                a["ldy"], a["res"], a["ldres"]) == want


@pytest.mark.parametrize("gate,up,want", [
    (dict(), None, ARG), (dict(), dict(dev=0x2000), ARG), (dict(), dict(fmt=0), FORMAT), (dict(fmt=2), dict(), FORMAT),
])
def test_pair_of_planes_refuses(gate, up, want):
    g, u = handle(**gate), handle(**up) if up is not None else None
    assert code("pgd_matrix_gemv_swiglu_mx_dev", C.byref(g), C.byref(u) if u is not None else None, A, 32, A, 16, 2, A,
                48) == want


@pytest.mark.parametrize("name,args,want", [
    ("pgd_matrix_upload_mxfp4", (A, None, A, 16, 32), ARG),
    ("pgd_matrix_upload_mxfp4", (None, A, A, 16, 32), ARG),
    ("pgd_matrix_from_mxfp4_dev", (A, None, 16, A, 16, 16, 32), ARG),
    ("pgd_matrix_from_mxfp4_dev", (A, A, 16, None, 16, 16, 32), ARG),
    ("pgd_matrix_from_mxfp4_dev", (A, A, 8, A, 16, 16, 32), SHAPE),
    ("pgd_matrix_from_mxfp4_dev", (A, A, 16, A, 4, 16, 32), SHAPE),
    ("pgd_matrix_from_mxfp4_dev", (A, A + 8, 16, A, 16, 16, 32), ARG),
    ("pgd_matrix_from_mxfp4_dev", (A, A, 16, A, 16, 0, 32), SHAPE),
    ("pgd_matrix_from_mxfp4_dev", (A, A, 16, A, 16, 16, 0), SHAPE),
    ("pgd_matrix_from_mxfp4_dev", (None, A, 16, A, 16, 16, 32), ARG),
    ("pgd_matrix_from_mxfp4_dev", (A, A, 32, A, 16, 16, 48), SHAPE),
    ("pgd_matrix_from_mxfp4_dev", (A, A, 16, A, 16, (1 << 30) + 1, 32), SHAPE),
    ("pgd_matrix_from_mxfp4_dev", (A, A, 1 << 30, A, 1 << 26, 16, (1 << 30) + 32), SHAPE),
    ("pgd_matrix_upload_mxfp4", (A, A, A, 16, 48), SHAPE),
    ("pgd_matrix_upload_mxfp4", (A, A, A, 0, 32), SHAPE),
    ("pgd_matrix_upload_mxfp4", (A, A, A, (1 << 30) + 1, 32), SHAPE),
])
def test_matrix_from_planes_refuses(name, args, want):
    out = C.c_void_p()
    assert code(name, *args, C.byref(out)) == want
    assert not out.value


def test_definition_rounds_to_the_nearest_code():
    """Every code is its own rounding, each middle goes to the even code, and 6 is the end."""
    x = np.zeros((1, 32), np.float32)
    x[0, :16] = mx.E2M1
    x[0, 16:23] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    x[0, 23:27] = [6.5, 7.0, -7.9, 0.2]
    c, s = mx.quantize(x)
    assert s[0, 0] == 127
    v = mx.values(c, s)[0]
    assert np.array_equal(v[:16], mx.E2M1)
    assert np.array_equal(v[16:23], [0, 1, 1, 2, 2, 4, 4]) and np.array_equal(v[23:27], [6, 6, -6, 0])


def test_definition_at_the_ends_of_the_range():
    x = np.zeros((5, 32), np.float32)
    x[1, 3] = np.float32(1e-45)
    x[2, 5] = np.finfo(np.float32).max
    x[3, 7], x[4, 9] = np.inf, np.nan
    c, s = mx.quantize(x)
    assert list(s[:, 0]) == [0, 0, 252, 255, 255]
    v = mx.values(c, s)
    assert not v[0].any() and not v[1].any() and v[2, 5] == 6 * 2.0 ** 125
    assert np.isnan(v[3]).all() and np.isnan(v[4]).all()


def test_other_activations_refuse_mxfp4():
    """Prepared A8 rows and paired quantized rows are for other formats."""
    m = handle()
    p = C.byref(m)
    assert code("pgd_matrix_gemv_act_dev", p, A, 1, A, 48, None, 0) == FORMAT
    assert code("pgd_matrix_gemv_act_dev_noalloc", p, A, 1, A, 48, None, 0) == FORMAT
    assert code("pgd_matrix_gemv_q8act_pair_dev", p, A, p, A, A, 64, 1, 48) == FORMAT
