"""The sizes of the MXFP4 tests take the kernels that they are there for (no GPU: the
library's choice is a function of sizes, types and strides)."""
import re
from pathlib import Path

import pytest

from mxfp4_choice import BF16, F16, F32, FEW, MANY, PLANES, choice, taken
from test_gpu_mxfp4_launches import LAUNCHES

# block shapes of the many-row kernel
SHAPES = {"planes": [(128, 256), (128, 128), (64, 128), (32, 128)], "terms": [(64, 256), (64, 128), (32, 128)],
          "digits": [(32, 256), (32, 128)]}


@pytest.mark.parametrize("case", MANY)
def test_size_takes_its_kernel(case):
    assert taken(*case) == MANY[case]


def test_every_block_shape_is_among_the_sizes():
    """Each shape alone and in ranges, for plain products and pairs (f32 terms of 64 rows and
    256 outputs in ranges are estimated slower than digits at every size)."""
    for kind, blocks in SHAPES.items():
        for block in blocks:
            for ranges in ("", "+"):
                for pair in (False, True):
                    if (kind, block, ranges, pair) == ("terms", (64, 256), "+", True):
                        continue
                    assert any(v == (kind, block, ranges) and c[4] == pair for c, v in MANY.items()), (kind, block, ranges, pair)


def test_launch_sizes_take_every_block_shape():
    seen = {(c.kind, c.block, c.ranges > 1) for c in (choice(t, n, k, rows) for t, n, k, rows in LAUNCHES)}
    want = {(kind, block, r) for kind, blocks in SHAPES.items() for block in blocks for r in (False, True)}
    assert want - seen == {("terms", (64, 128), True)}  # (among MANY)


def test_few_rows_and_captures():
    """What a stream capture refuses is what needs scratch memory; few rows split themselves."""
    for t, most in ((F32, 5), (F16, 8), (BF16, 4)):
        assert choice(t, 48, 96, most, scratch=False).kind == "rows"
        assert choice(t, 48, 96, most + 1, scratch=False).prep
    assert choice(BF16, 48, 128, 900, scratch=False) == ("terms", (), 1, False)
    for rows in (1, 16, 47, 333, 4000):
        c = choice(PLANES, 5120, 4096, rows, scratch=False)
        assert c.ranges == 1 and not c.prep


def test_few_sizes_take_the_few_row_kernel():
    got = [choice(*c) for c in FEW]
    assert all(not c.block for c in got) and {c.kind for c in got} == {"rows", "terms", "planes"}


def test_f32_rows_are_exact_up_to_16():
    for n, k in ((40, 96), (1000, 512), (5120, 17408), (17408, 5120), (151936, 896)):
        for pair in (False, True):
            assert all(choice(F32, n, k, rows, pair).kind in ("terms", "rows") for rows in range(1, 17))
    assert choice(F32, 5120, 17408, 17).kind == "digits"


def test_long_strides_stay_in_the_few_row_kernel():
    """The many-row kernel's lanes hold offsets in 32 bits."""
    assert choice(BF16, 2100, 512, 1100, stride=(1 << 24) - 16).block
    assert not choice(BF16, 2100, 512, 1100, stride=1 << 24).block
    assert not choice(PLANES, 5008, 160, 1300, stride=1 << 24).block


def test_launches_stay_below_2_32_threads():
    """The largest matrices and most rows: the many-row kernel's workgroups of 256 threads, and
    the digits' (two tiles of 16 rows by 128 columns each), fit one launch of HIP."""
    for n, k, rows in ((1 << 30, 32, 65), (1 << 30, 32, 129), (1 << 30, 128, 4096), (1 << 24, 64, 1 << 20),
                       (4096, 128, (1 << 31) - 1), (151936, 896, 1 << 26), (32, 1 << 24, 4096), (32, 1 << 23, 8192)):
        for t in (F32, F16, BF16, PLANES):
            for pair in (False, True):
                if pair and t in (F16, BF16):
                    continue
                c = choice(t, n, k, rows, pair)
                if c.block:
                    outs = -(-n // 16) * 16 * (2 if pair else 1)
                    blocks = -(-rows // c.block[0]) * -(-outs // c.block[1]) * c.ranges
                    assert -(-blocks // 8) * 8 * 256 < 1 << 32, (t, n, k, rows, pair, c)
                if c.kind == "digits":
                    assert -(-rows // 16) * -(-k // 128) // 2 * 256 < (1 << 32) - 256, (n, k, rows)
