"""Which kernel an MXFP4 product takes: the library's own choice (host only), and sizes
that take each block shape of the many-row kernel, with and without ranges of k tiles and
with a last k tile that is not whole."""
import ctypes as C
from typing import NamedTuple

F32, F16, BF16, PLANES = 0, 1, 2, 3
KINDS = ("planes", "terms", "digits", "rows")


class _Many(C.Structure):
    _fields_ = [("shape", C.c_int), ("ranges", C.c_int), ("block_rows", C.c_int), ("block_outs", C.c_int), ("us", C.c_double)]


class _Choice(C.Structure):
    _fields_ = [("kind", C.c_int), ("prep", C.c_bool), ("few", C.c_bool), ("many", _Many)]


class Choice(NamedTuple):
    kind: str    # how the rows are held
    block: tuple  # rows and outputs of a block; () in the few-row kernel
    ranges: int  # of k tiles
    prep: bool   # rows are split into scratch memory first


def choice(t: int, n: int, k: int, rows: int, pair: bool = False, scratch: bool = True, stride: int = 0) -> Choice:
    """For rows of a type (stride in bytes; 0: rows without gaps)."""
    from pagoda_amd import _lib

    f = _lib.lib()["_ZN3pgd2mx6chooseEiibixib"]  # pgd::mx::choose
    f.restype = _Choice
    f.argtypes = [C.c_int, C.c_int, C.c_bool, C.c_int, C.c_longlong, C.c_int, C.c_bool]
    c = f(n, k, pair, t, stride or {F32: 4 * k, F16: 2 * k, BF16: 2 * k, PLANES: k // 2}[t], rows, scratch)
    block = () if c.few else (c.many.block_rows, c.many.block_outs)
    return Choice(KINDS[c.kind], block, 1 if c.few else c.many.ranges, c.prep)


# (type, outputs, width, rows, pair) -> kind and block; "+": in ranges of k tiles
MANY = {
    (F32, 2100, 416, 500, False): ("digits", (32, 256), ""),
    (F32, 1300, 4128, 100, False): ("digits", (32, 256), "+"),
    (F32, 330, 544, 500, False): ("digits", (32, 128), ""),
    (F32, 40, 2080, 900, False): ("digits", (32, 128), "+"),
    (F32, 520, 416, 900, True): ("digits", (32, 256), ""),
    (F32, 200, 4128, 333, True): ("digits", (32, 256), "+"),
    (F32, 330, 544, 500, True): ("digits", (32, 128), ""),
    (F32, 200, 6176, 65, True): ("digits", (32, 128), "+"),
    (F32, 2100, 160, 1100, False): ("terms", (64, 256), ""),
    (F32, 2100, 160, 500, False): ("terms", (64, 128), ""),
    (F32, 1300, 160, 130, False): ("terms", (32, 128), ""),
    (F32, 40, 4128, 17, False): ("terms", (32, 128), "+"),
    (F32, 2100, 160, 500, True): ("terms", (64, 256), ""),
    (F32, 520, 160, 900, True): ("terms", (64, 128), ""),
    (F32, 2100, 2080, 33, True): ("terms", (64, 128), "+"),
    (F32, 1300, 160, 130, True): ("terms", (32, 128), ""),
    (F32, 40, 4128, 17, True): ("terms", (32, 128), "+"),
    (F16, 2100, 160, 1100, False): ("terms", (64, 256), ""),
    (F16, 1300, 6176, 200, False): ("terms", (64, 256), "+"),
    (F16, 2100, 160, 500, False): ("terms", (64, 128), ""),
    (F16, 40, 8224, 333, False): ("terms", (64, 128), "+"),
    (F16, 2100, 160, 65, False): ("terms", (32, 128), ""),
    (F16, 40, 2080, 33, False): ("terms", (32, 128), "+"),
    (BF16, 2100, 160, 1100, False): ("terms", (64, 256), ""),
    (BF16, 2100, 512, 1100, False): ("terms", (64, 256), ""),
    (BF16, 2100, 4096, 500, False): ("terms", (64, 256), "+"),
    (BF16, 2100, 512, 500, False): ("terms", (64, 128), ""),
    (BF16, 40, 6176, 1100, False): ("terms", (64, 128), "+"),
    (BF16, 1300, 512, 65, False): ("terms", (32, 128), ""),
    (BF16, 40, 4096, 20, False): ("terms", (32, 128), "+"),
    (PLANES, 5008, 160, 1300, False): ("planes", (128, 256), ""),
    (PLANES, 2100, 8224, 1100, False): ("planes", (128, 256), "+"),
    (PLANES, 2100, 160, 1100, False): ("planes", (128, 128), ""),
    (PLANES, 5008, 8224, 65, False): ("planes", (128, 128), "+"),
    (PLANES, 2100, 160, 500, False): ("planes", (64, 128), ""),
    (PLANES, 40, 8224, 333, False): ("planes", (64, 128), "+"),
    (PLANES, 5008, 160, 65, False): ("planes", (32, 128), ""),
    (PLANES, 40, 4128, 47, False): ("planes", (32, 128), "+"),
    (PLANES, 3300, 160, 900, True): ("planes", (128, 256), ""),
    (PLANES, 2100, 8224, 500, True): ("planes", (128, 256), "+"),
    (PLANES, 2100, 160, 500, True): ("planes", (128, 128), ""),
    (PLANES, 2100, 8224, 65, True): ("planes", (128, 128), "+"),
    (PLANES, 520, 160, 900, True): ("planes", (64, 128), ""),
    (PLANES, 200, 8224, 65, True): ("planes", (64, 128), "+"),
    (PLANES, 3300, 160, 65, True): ("planes", (32, 128), ""),
    (PLANES, 40, 4128, 47, True): ("planes", (32, 128), "+"),
}

# The few-row kernel: rows split inside the launch, terms and planes in 1 to 4 row tiles.
FEW = [(F32, 333, 416, 1, False), (F32, 333, 416, 5, True), (F32, 100, 896, 16, False), (F32, 100, 160, 40, True),
       (F16, 333, 416, 8, False), (F16, 100, 160, 20, False), (F16, 100, 160, 70, False), (BF16, 333, 416, 4, False),
       (BF16, 100, 160, 40, False), (PLANES, 333, 416, 9, False), (PLANES, 100, 160, 40, True), (PLANES, 100, 160, 70, False)]


def taken(t: int, n: int, k: int, rows: int, pair: bool) -> tuple:
    c = choice(t, n, k, rows, pair)
    return c.kind, c.block, "+" if c.ranges > 1 else ""
