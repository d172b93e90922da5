"""The 8-bit paged KV cache in NumPy, from its definition: e4m3 codes as the multiples of
their step, pages in float64, attention in float64 with the bound on what f32 sums and the
roundings of each type may be off."""
import numpy as np

PAGE = 16
F32, F16, BF16 = 0, 1, 2
SIZES = {F32: 4, F16: 2, BF16: 2}


# ---- row types -------------------------------------------------------------------


def bf16_bits(x):
    """f32 to bf16 bits, to nearest, ties to even (infinities stay, NaN becomes a quiet one)."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((b.astype(np.uint64) + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where((b & 0x7FFFFFFF) > 0x7F800000, np.uint16(0x7FC0), r)


def bf16_value(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def typed(x, t):
    """f32 values as rows of a type: what a call takes, and their values in float64."""
    x = np.ascontiguousarray(x, np.float32)
    if t == F32:
        return x, x.astype(np.float64)
    if t == F16:
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h, h.astype(np.float64)
    b = bf16_bits(x)
    return b, bf16_value(b).astype(np.float64)


def value(raw, t):
    return (bf16_value(raw) if t == BF16 else raw).astype(np.float64)


def half_step(t):
    return {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[t]


# ---- codes and pages ---------------------------------------------------------------


def round_e4m3(u):
    """float64 of magnitude up to 448 to the nearest e4m3 value, ties to the even one."""
    u = np.asarray(u, np.float64)
    _, e = np.frexp(np.abs(u))
    step = np.ldexp(1.0, np.maximum(e - 4, -9))
    return np.rint(u / step) * step


def holds(top, most=448.0):
    """Smallest e >= -126 with top <= most * 2^e."""
    m, e = np.frexp(np.float64(top) / most)
    return max(int(e) - (1 if m == 0.5 else 0), -126) if top > 0 else -126


class Cache:
    """Pages as units (code values) [pages, kv, 16, hd], exponents [pages, kv] of K (0) and V (1), NaN places."""

    def __init__(self, n_pages, kv, hd):
        self.n, self.kv, self.hd = n_pages, kv, hd
        self.units = np.zeros((2, n_pages, kv, PAGE, hd))
        self.exps = np.full((2, n_pages, kv), -126)
        self.nan = np.zeros((n_pages, kv, PAGE), bool)
        self.filled = np.zeros(n_pages, int)

    def append(self, k, v, slots):
        """float64 rows [rows, kv * hd] in the order of their slots."""
        row = 0
        slots = [int(s) for s in slots]
        while row < len(slots):
            first, n = slots[row], 1
            if not 0 <= first < self.n * PAGE:
                row += 1
                continue
            while row + n < len(slots) and slots[row + n] == first + n and (first + n) % PAGE:
                n += 1
            self._page(first // PAGE, first % PAGE, [x[row:row + n].reshape(n, self.kv, self.hd) for x in (k, v)])
            row += n

    def _page(self, page, s0, rows):
        n = rows[0].shape[0]
        for h in range(self.kv):
            bad = ~(np.isfinite(rows[0][:, h]).all(1) & np.isfinite(rows[1][:, h]).all(1))
            self.nan[page, h, s0:] = False
            if s0 == 0:
                self.nan[page, h] = False
            self.nan[page, h, s0:s0 + n] = bad
            for w in range(2):
                x = np.where(bad[:, None], 0.0, rows[w][:, h])
                e0 = self.exps[w, page, h] if s0 else -126
                e = max(e0, holds(np.abs(x).max()))
                old = round_e4m3(self.units[w, page, h, :s0] * 2.0 ** (e0 - e))
                self.units[w, page, h] = 0
                self.units[w, page, h, :s0] = old
                self.units[w, page, h, s0:s0 + n] = round_e4m3(x * 2.0 ** -e)
                self.exps[w, page, h] = e
        self.filled[page] = s0 + n

    def values(self, w):
        """[pages, kv, 16, hd], NaN where an entry's row had a non-finite value."""
        x = self.units[w] * 2.0 ** self.exps[w].astype(np.float64)[..., None, None]
        return np.where(self.nan[..., None], np.nan, x)

    def read(self, w, slots):
        s = np.asarray(slots)
        return self.values(w)[s // PAGE, :, s % PAGE].reshape(len(s), -1)

    def bounds(self, page):
        """hi, lo [kv, hd] of the key codes in steps of 4, outward."""
        u = self.units[0, page, :, :max(self.filled[page], 1)]
        return np.ceil(u.max(1) / 4), np.floor(u.min(1) / 4)


# ---- a step's sequences ----------------------------------------------------------------


def pages(n):
    return -(-n // PAGE)


class Step:
    """Sequences of given contexts and row counts over a cache of random pages in random order."""

    def __init__(self, rng, kv, hd, ctx, new, t, spare=3, widen=2, scale=1.0):
        self.ctx, self.new, self.t = list(ctx), list(new), t
        need = [pages(c) for c in ctx]
        self.cache = Cache(sum(need) + spare, kv, hd)
        order = rng.permutation(self.cache.n)
        self.width = max(need + [1]) + widen
        self.tables = np.full((len(ctx), self.width), -7, np.int32)
        at, slots = 0, []
        for s, (c, m) in enumerate(zip(ctx, need)):
            self.tables[s, :m] = order[at:at + m]
            at += m
            p = np.arange(c)
            slots.append(self.tables[s, p // PAGE] * PAGE + p % PAGE)
        self.slots = np.concatenate(slots + [np.zeros(0, int)]).astype(np.int32)
        size = np.exp(rng.normal(0, 0.7, kv * hd)) * scale
        rows = rng.normal(0, 1, (2, len(self.slots), kv * hd)) * 2.0 ** rng.integers(-3, 4, (2, len(self.slots), 1))
        (self.k_raw, k), (self.v_raw, v) = typed(rows[0] * size, t), typed(rows[1], t)
        self.cache.append(k, v, self.slots)
        self.row_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.row_start[-1])
        self.lens = np.array(ctx, np.int32)

    def each_row(self):
        """(row, sequence, positions seen)"""
        for s, (c, n) in enumerate(zip(self.ctx, self.new)):
            for j in range(n):
                yield int(self.row_start[s]) + j, s, max(c - n + j + 1, 0)


def attend(q, k, v, t, unit=0.0):
    """One query [hd] over positions k, v [n, hd] (float64): the result and the bound on what a kernel with f32
    sums may be off. unit: the power of two of each position's value codes.

    A score of hd products in at most two terms, summed in any order, q held to 2^-22: (3 hd + 4) 2^-23 of
    sum |q k|, and one rounding of the scaled score, of its maximum's difference and
    of the exponent's argument, each 2^-24 of its magnitude, 2^-22 for exp2 itself. Weights then
    are off by the factor exp(2 d). They enter as f16 terms of 11 bits: one (bf16 rows) to nearest is 2^-11
    off at most; of two the first is truncated, 2^-10, and the second to nearest, 2^-11 of that; and no
    less than f16's smallest half step, 2^-25, times 2^-11 the weights' scale: 2^-36 of a weight that is the
    largest or up to 2^4 below; codes are up to 448. The sums of n weights and n products by n 2^-23 each."""
    if len(k) == 0:
        return np.zeros(v.shape[1]), np.zeros(v.shape[1])
    hd = k.shape[1]
    s = k @ q / np.sqrt(hd)
    if not np.isfinite(s).all() or not np.isfinite(v).all():
        return np.full(hd, np.nan), np.zeros(hd)
    d = ((3 * hd + 4) * 2.0 ** -23 * (np.abs(k) @ np.abs(q)).max() / np.sqrt(hd)
         + 4 * 2.0 ** -24 * 1.5 * np.abs(s).max() + 2.0 ** -22)
    w = np.exp(s - s.max())
    w /= w.sum()
    held = {F32: 2.0 ** -21, F16: 2.0 ** -21, BF16: 2.0 ** -11}[t]
    mass = w @ np.abs(v)
    small = len(k) * 448 * 2.0 ** -36 * (w * unit).max()
    return w @ v, mass * (2 * np.expm1(2 * d) + held + (2 * len(k) + 16) * 2.0 ** -23) + small


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-x))


def attention(step, q, t, heads, gate=None, picked=None):
    """float64 results [rows, heads, hd] and their bounds; picked: (row, kv head) -> places in the table."""
    c = step.cache
    g = heads // c.kv
    out, bound = np.zeros((step.rows, heads, c.hd)), np.zeros((step.rows, heads, c.hd))
    kv = [c.values(w) for w in range(2)]
    for row, s, seen in step.each_row():
        for h in range(heads):
            head = h // g
            places = np.arange(pages(seen)) if picked is None else np.asarray(picked[row][head], int)
            at = (places[:, None] * PAGE + np.arange(PAGE)).reshape(-1)
            use = at < seen
            kk, vv = (x[step.tables[s, places], head].reshape(-1, c.hd)[use] for x in kv)
            unit = 2.0 ** c.exps[1, step.tables[s, places], head].astype(float).repeat(PAGE)[use]
            o, b = attend(q[row, h], kk, vv, t, unit)
            if gate is not None:
                sg = sigmoid(gate[row, h])
                # sigmoid: exp2 of a rounded product, a sum, a quotient; then the product
                b = b * sg + np.abs(o) * sg * (8 + 2 * np.abs(gate[row, h])) * 2.0 ** -24
                o = o * sg
            out[row, h] = o
            bound[row, h] = b + np.abs(o) * half_step(t) * 1.01 + 2.0 ** -140 + (2.0 ** -24 if t == F16 else 0)
    return out, bound


def select(step, q, heads, top, sinks, recent):
    """row -> KV head -> chosen places, ascending; from the scores as whole numbers."""
    c = step.cache
    g = heads // c.kv
    bounds = [c.bounds(p) for p in range(c.n)]
    out = {}
    for row, s, seen in step.each_row():
        out[row] = []
        n = min(pages(seen), step.width)
        for head in range(c.kv):
            qs = q[row, head * g:(head + 1) * g]
            qs = np.where(np.isfinite(qs), qs, 0.0)
            q8 = np.rint(qs * 2.0 ** -holds(np.abs(qs).max(), 127.0)).astype(np.int64)
            score = []
            for p in step.tables[s, :n]:
                if not 0 <= p < c.n:
                    score.append(-np.inf)
                    continue
                hi, lo = (b[head].astype(np.int64) for b in bounds[p])
                best = max(int(np.maximum(x * hi, x * lo).sum()) for x in q8)
                with np.errstate(over="ignore"):
                    score.append(float(np.float32(best) * np.float32(2.0 ** int(c.exps[0, p, head]))))
            order = sorted(range(n), key=lambda p: (not (p < sinks or p >= n - recent), -score[p], p))
            out[row].append(sorted(order[:top]))
    return out
