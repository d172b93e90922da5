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


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_attention(heads, kv, hd):
    size = lambda nseq, blocks, rows, most: lib().pgd_attn_kv8_rows_ws_bytes(heads, kv, hd, nseq, blocks, rows, most)
    for nseq, blocks in ((1, 100), (7, 600), (64, 8200)):
        for most in (0, 1, 3, 22, 100, 5000):
            never_falls(lambda r: size(nseq, blocks, r, most), ROWS)
        for rows in ROWS:
            never_falls(lambda m: size(nseq, blocks, rows, m), [0] + ROWS)
            assert size(nseq, blocks, rows, rows) == size(nseq, blocks, rows, 2 ** 31 - 1)
            assert size(nseq, blocks, rows, rows) == lib().pgd_attn_kv8_ws_bytes(heads, kv, hd, nseq, blocks, rows)
    for rows in ROWS:
        never_falls(lambda n: size(n, 600, rows, 4), [1, 2, 31, 32, 33, 64, 65, 1000])
        never_falls(lambda b: size(40, b, rows, 4), BLOCKS)
    assert size(1, 100, 8, -1) == 0 == size(1, 100, -8, 1)


def test_decode_steps_need_no_prompts_workspace():
    """At most 2.25 partial sums (16 queries of a head, with their two maxima and sum) per workgroup that runs at once, 32 bytes
    a row beside them: of one row, whatever max_rows says, and of more rows by max_rows."""
    most = 2.25 * 512 * 16 * (256 + 4) * 4
    assert 0 < lib().pgd_attn_kv8_ws_bytes(24, 4, 256, 1, 8200, 1) <= most + 32
    assert 0 < lib().pgd_attn_kv8_rows_ws_bytes(24, 4, 256, 32, 8200, 32, 1) <= most + 32 * 32


def test_the_most_rows_that_a_launch_holds():
    """Four results of a row and head a workgroup of 256 threads, below 2^32 threads: the sizes past that are refused."""
    for size in (lambda rows: lib().pgd_attn_kv8_ws_bytes(1, 1, 64, 2, 40, rows),
                 lambda rows: lib().pgd_attn_kv8_ws_bytes(2, 1, 64, 2, 40, rows // 2)):
        assert size(2 ** 26 - 4) > 0
        for rows in (2 ** 26 - 2, 2 ** 26, 2 ** 26 + 2):
            assert size(rows) == 0
    assert lib().pgd_attn_kv8_ws_bytes(1, 1, 64, 2, 40, 2 ** 26 - 3) == 0 == lib().pgd_attn_kv8_ws_bytes(1, 1, 64, 2, 40, 2 ** 26 - 1)
