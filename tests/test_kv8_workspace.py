"""Workspaces of the 8-bit KV cache's attention on the host: one that is large enough for a step is large enough for
every smaller one."""
import pytest

SHAPES = [(24, 4, 256), (14, 2, 64), (28, 4, 128), (40, 2, 128), (3, 3, 256), (34, 1, 64)]
ROWS = [1, 2, 3, 5, 8, 17, 24, 31, 32, 33, 60, 95, 96, 97, 127, 128, 129, 192, 255, 256, 257, 511, 512, 1000, 5000]
BLOCKS = [1, 15, 16, 17, 18, 24, 25, 40, 100, 600, 601, 8200, 100000]
TOPS = [1, 8, 15, 16, 17, 23, 24, 25, 33, 64, 100, 127, 128, 129, 200, 1000, 3000]


def lib():
    from pagoda_amd import _lib

    return _lib.lib()


def never_falls(f, values):
    got = [f(v) for v in values]
    assert got == sorted(got), list(zip(values, got))


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_lists(heads, kv, hd):
    size = lambda rows, blocks, top: lib().pgd_kv8_sparse_ws_bytes(heads, kv, hd, rows, blocks, top)
    for blocks in (17, 600, 8200):
        for top in TOPS:
            never_falls(lambda r: size(r, blocks, top), ROWS)
        for rows in ROWS:
            never_falls(lambda t: size(rows, blocks, t), TOPS)
    for rows in ROWS:
        for top in TOPS:
            never_falls(lambda b: size(rows, b, top), BLOCKS)
    # the scores, and partial sums of at most twice as many pieces of lists as run at once
    assert size(32, 600, 128) <= max(32 * kv * 600 * 4, 2 * 1024 * 16 * (hd + 4) * 4)
