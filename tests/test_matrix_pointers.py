"""Device addresses of the Python layer are whole numbers: host memory (bytes, strings, arrays,
which ctypes would pass by address) never reaches the library. Without a GPU: what is taken
is refused by the library's own checks before the first HIP call."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest

from test_mxfp4_host import A, ARG, SHAPE, handle

HOST = [b"rows", "rows", (C.c_char * 64)(), np.zeros(4), 4096.0, C.c_void_p(A)]


def calls():
    """name, the call with its device addresses left open, how many, the code that sane ones get."""
    from pagoda_amd import Matrix
    from pagoda_amd.matrix import mxfp4_quantize_dev

    structs = handle(fmt=1), handle(fmt=5)
    q4k, mx = (Matrix.__new__(Matrix) for _ in structs)
    q4k.handle, mx.handle = (C.c_void_p(C.addressof(s)) for s in structs)
    q4k.keep, mx.keep = structs
    q4k.free = mx.free = lambda: None  # (nothing to free behind these handles)
    dev = SimpleNamespace(handle=None)
    return [
        ("gemv_dev", lambda x, y, res: q4k.gemv_dev(x, 64, 2, y, 40, False, res, 48), 3, SHAPE),
        ("gemv_swiglu_dev", lambda x, y: Matrix.gemv_swiglu_dev(q4k, q4k, x, 64, 2, y, 40), 2, SHAPE),
        ("gemv_mx_dev", lambda c, s, y, res: mx.gemv_mx_dev(c, 32, s, 16, 2, y, 40, res, 48), 4, SHAPE),
        ("gemv_swiglu_mx_dev", lambda c, s, y: Matrix.gemv_swiglu_mx_dev(mx, mx, c, 32, s, 16, 2, y, 40), 3, SHAPE),
        ("mxfp4_quantize_dev", lambda x, c, s, v: mxfp4_quantize_dev(dev, x, 0, 64, 2, 64, c, 32, s, 16, v, 64), 4, ARG),
    ]


@pytest.mark.parametrize("which", range(5))
def test_host_memory_is_no_device_address(which):
    from pagoda_amd import PagodaError

    name, call, count, code = calls()[which]
    for good in (A, np.int64(A), np.uint64(A)):
        with pytest.raises(PagodaError) as e:
            call(*[good] * count)
        assert e.value.code == code, name
    for i in range(count):
        for bad in HOST:
            if isinstance(bad, np.ndarray):
                bad = bad.copy()
            args = [A] * count
            args[i] = bad
            with pytest.raises((TypeError, ValueError)):
                call(*args)


def test_none_is_a_null_pointer():
    from pagoda_amd import PagodaError

    for name, call, count, _ in calls():
        with pytest.raises(PagodaError) as e:
            call(*[None] * count)
        assert e.value.code == ARG, name
