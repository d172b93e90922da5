"""MXFP4 in NumPy, from the format's definition: what the GPU tests compare with."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], np.float64)


def quantize(x: np.ndarray):
    """float32 rows [rows, k] -> codes u8 [rows, k / 2], scales u8 [rows, k / 32]. Every
    code is the nearest of the eight magnitudes by comparison in float64, the even one on ties."""
    rows, k = x.shape
    b = x.reshape(rows, k // 32, 32)
    bits = b.view(np.uint32) & 0x7FFFFFFF
    e = (bits.max(-1) >> 23).astype(np.int64)
    scales = np.where(e == 255, 255, np.maximum(e - 2, 0)).astype(np.uint8)
    with np.errstate(invalid="ignore", over="ignore"):
        v = np.abs(b.astype(np.float64)) * 2.0 ** (127.0 - scales.astype(np.float64))[..., None]
    code = np.zeros(b.shape, np.uint8)
    for c in range(7):  # between code c and c + 1: up past the middle, on it if c + 1 is even
        mid = (E2M1[c] + E2M1[c + 1]) / 2
        code += (v >= mid if c % 2 else v > mid).astype(np.uint8)
    code |= (b.view(np.uint32) >> 31).astype(np.uint8) << 3
    code[scales == 255] = 0
    code = code.reshape(rows, k)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """float64 values [rows, k] of planes (row strides may exceed the rows)."""
    rows = codes.shape[0]
    c = np.stack([codes & 15, codes >> 4], -1).reshape(rows, -1)
    nblk = c.shape[1] // 32
    with np.errstate(invalid="ignore"):
        s = np.where(scales[:, :nblk] == 255, np.nan, 2.0 ** (scales[:, :nblk].astype(np.float64) - 127.0))
        return (E2M1[c].reshape(rows, nblk, 32) * s[..., None]).reshape(rows, -1)


def bf16(x: np.ndarray) -> np.ndarray:
    """float32 -> bf16 bits (u16), nearest even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_f32(h: np.ndarray) -> np.ndarray:
    return (h.astype(np.uint32) << 16).view(np.float32)


def rows_of(x: np.ndarray, t: int):
    """Rows as type t (0 f32, 1 f16, 2 bf16): what is uploaded, and its value in float32."""
    if t == 0:
        return x, x
    if t == 1:
        h = x.astype(np.float16)
        return h, h.astype(np.float32)
    h = bf16(x)
    return h, bf16_f32(h)


def padded(a: np.ndarray, ld: int, fill) -> np.ndarray:
    """Rows of stride ld, the gap holding `fill`."""
    out = np.full((a.shape[0], ld), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


def product_bound(x: np.ndarray, w: np.ndarray) -> np.ndarray:
    """How far f32 sums of the exact products x w^T may be off: one rounding
    (at most 2^-23 of the running sum, should the hardware truncate) per
    addition, k + 32 of them at most with the joins of partial sums, against
    the sum of magnitudes; plus the smallest normal number for results below it."""
    k = x.shape[1]
    return (k + 32) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T) + 2.0 ** -126


def silu(g: np.ndarray) -> np.ndarray:
    return g / (1.0 + np.exp(-g))


def swiglu_bound(x: np.ndarray, wg: np.ndarray, wu: np.ndarray) -> np.ndarray:
    """silu' is at most 1.1 and |silu(g)| <= |g|; the epilogue's exp, division and
    product add under 8 roundings of 2^-23 of the result."""
    g, u = x @ wg.T, x @ wu.T
    dg, du = product_bound(x, wg), product_bound(x, wu)
    return 1.1 * dg * (np.abs(u) + du) + (np.abs(silu(g)) + 1.1 * dg) * du + 2.0 ** -20 * np.abs(silu(g) * u) + 2.0 ** -126
