"""Timed cases of the 8-bit paged KV cache: block tables built on the GPU, the
write, attention over it, and attention over the pages a cheap score selects.

A page holds 16 positions of every KV head. A (page, KV head) has one power of
two 2^e for its keys and one for its values; an entry is an e4m3 code (sign, 4
exponent bits, 3 mantissa bits, largest 448) times that. e is the smallest
exponent that holds the page's largest magnitude; while a page fills it never
falls, and when it grows the codes already there are rounded again. Per page,
KV head and channel two whole numbers bound the keys' codes from above and below in
steps of 4. Kinds of case (`kind`):

  tables  a step's bookkeeping: pages from the free list into the block tables,
          and the row starts, sequences, positions and slots of the new rows.
  write   a step's K and V rows into their pages, and the pages' positions read
          back.
  attn    causal attention of the rows over their sequences' pages, with or
          without the sigmoid gate.
  sparse  per (row, KV head) the pages with the highest bounds on q.k (of q in
          8 bits; the first and the latest pages always), and attention over those.

Contexts and row counts are spread geometrically over a case's sequences, in an
order that the seed gives; pages lie in the pool in random order. Keys
have channels of different sizes, as projections leave them.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 16
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 2}
_FREE_SPARE = 64  # pages on the free list beyond those that a step takes


def listed() -> list[dict]:
    return [
        # one user's next token: the smallest step
        {"name": "tables_1", "kind": "tables", "nseq": 1, "shortest": 80, "longest": 80, "few": 1, "tokens": 1},
        # a full server: most requests decode, some bring prompts
        {"name": "tables_512", "kind": "tables", "nseq": 512, "shortest": 1, "longest": 8000, "few": 1, "tokens": 500},
        # one decoded token of the 0.5B model into a page that is half full
        {"name": "write_1", "kind": "write", "kv_heads": 2, "head_dim": 64, "nseq": 1, "shortest": 88, "longest": 88,
         "few": 1, "tokens": 1, "type": "f32"},
        # a few prompts of the 27B-class model, behind short cached prefixes
        {"name": "write_prompts", "kind": "write", "kv_heads": 4, "head_dim": 256, "nseq": 5, "shortest": 3,
         "longest": 60, "few": 333, "tokens": 4096, "type": "bf16"},
        # attention of one decoded token after a chat prompt on the 0.5B model
        {"name": "attn_1", "kind": "attn", "heads": 14, "kv_heads": 2, "head_dim": 64, "nseq": 1, "shortest": 81,
         "longest": 81, "few": 1, "tokens": 1, "type": "f32", "gate": False},
        # a served batch of the 27B-class model, contexts over two decades
        {"name": "attn_32", "kind": "attn", "heads": 24, "kv_heads": 4, "head_dim": 256, "nseq": 32, "shortest": 40,
         "longest": 4000, "few": 1, "tokens": 1, "type": "f32", "gate": True},
        # four proposed tokens a request are verified
        {"name": "attn_verify_16", "kind": "attn", "heads": 24, "kv_heads": 4, "head_dim": 256, "nseq": 16,
         "shortest": 100, "longest": 6000, "few": 4, "tokens": 4, "type": "f16", "gate": True},
        # long documents: the cache is most of what is read
        {"name": "attn_long_8", "kind": "attn", "heads": 28, "kv_heads": 4, "head_dim": 128, "nseq": 8,
         "shortest": 20000, "longest": 130000, "few": 1, "tokens": 1, "type": "bf16", "gate": False},
        # prompt chunks behind cached prefixes
        {"name": "attn_prompts", "kind": "attn", "heads": 24, "kv_heads": 4, "head_dim": 256, "nseq": 3,
         "shortest": 500, "longest": 4001, "few": 211, "tokens": 1500, "type": "f32", "gate": False},
        # one user's long document, a sixteenth of it read
        {"name": "sparse_1", "kind": "sparse", "heads": 24, "kv_heads": 4, "head_dim": 256, "nseq": 1,
         "shortest": 32777, "longest": 32777, "few": 1, "tokens": 1, "type": "f32", "gate": True, "top": 128,
         "sinks": 1, "recent": 2},
        # a served batch of long contexts
        {"name": "sparse_24", "kind": "sparse", "heads": 28, "kv_heads": 4, "head_dim": 128, "nseq": 24,
         "shortest": 3000, "longest": 60000, "few": 1, "tokens": 1, "type": "bf16", "gate": False, "top": 64,
         "sinks": 1, "recent": 2},
        # two proposed tokens a request on middling contexts
        {"name": "sparse_verify_9", "kind": "sparse", "heads": 16, "kv_heads": 2, "head_dim": 256, "nseq": 9,
         "shortest": 30, "longest": 9000, "few": 2, "tokens": 2, "type": "f16", "gate": True, "top": 50, "sinks": 2,
         "recent": 4},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["tables", "write", "attn", "attn", "attn", "sparse", "sparse"])
    if kind == "tables":
        lo, few = _log(rng, 1, 500), rng.choice([1, 1, rng.randint(0, 4)])
        return {"kind": kind, "nseq": _log(rng, 1, 512), "shortest": lo, "longest": _log(rng, lo, 8000), "few": few,
                "tokens": _log(rng, max(few, 1), 500)}
    heads, kv, hd = rng.choice([(24, 4, 256), (14, 2, 64), (16, 2, 256), (28, 4, 128)])
    case = {"kind": kind, "kv_heads": kv, "head_dim": hd, "type": rng.choice(sorted(_TYPES))}
    if kind == "write":
        lo, few = rng.randint(0, 40), _log(rng, 1, 300)
        nseq = _log(rng, 1, 64)
        return {**case, "nseq": nseq, "shortest": lo, "longest": rng.randint(lo, 100), "few": few,
                "tokens": _log(rng, few, max(few, 4096 // nseq))}
    case.update(heads=heads, gate=rng.random() < 0.5)
    if kind == "sparse":
        nseq, lo, few = _log(rng, 1, 24), _log(rng, 20, 5000), rng.choice([1, 1, 1, 3])
        sinks, recent = rng.randint(0, 2), rng.randint(1, 4)
        return {**case, "nseq": nseq, "shortest": lo, "longest": _log(rng, lo, 60000), "few": few, "tokens": few,
                "top": _log(rng, 8, 200), "sinks": sinks, "recent": recent}
    if rng.random() < 0.7:  # decode and verify batches
        nseq, lo, few = _log(rng, 1, 64), _log(rng, 16, 1000), rng.choice([1, 1, 4])
        return {**case, "nseq": nseq, "shortest": lo, "longest": _log(rng, lo, min(130000, 500000 // nseq)), "few": few,
                "tokens": few}
    nseq, few = rng.randint(1, 3), _log(rng, 5, 400)
    tokens = _log(rng, few, 1200)
    return {**case, "nseq": nseq, "shortest": few, "longest": _log(rng, max(few, 300), 4000), "few": few,
            "tokens": tokens}


# ---- inputs -------------------------------------------------------------------


def _gen(seed: int, stream: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1_000_003 + stream) & 0x7FFFFFFFFFFFFFFF)
    return g


def _normal(shape, seed: int, stream: int) -> torch.Tensor:
    return torch.randn(shape, generator=_gen(seed, stream), device="cuda")


def _spread(lo: int, hi: int, n: int, seed: int, stream: int) -> list[int]:
    """n whole numbers from lo to hi in geometric steps, in the seed's order."""
    if n == 1:
        return [hi]
    order = torch.randperm(n, generator=torch.Generator().manual_seed(int(seed) * 31 + stream)).tolist()
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1)))) - 1 for i in order]


def _pages(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _geometry(case: dict, seed: int):
    """Per sequence: positions before the step's rows, and the number of rows."""
    n = case["nseq"]
    ctx = _spread(case["shortest"], case["longest"], n, seed, 1)
    new = _spread(case["few"], case["tokens"], n, seed, 2)
    if case["kind"] in ("attn", "sparse"):  # contexts with the rows in them
        return [max(c - t, 0) for c, t in zip(ctx, new)], new
    return ctx, new


def _step_inputs(case: dict, seed: int) -> dict:
    """A step's host-known sizes and its device arrays: lengths before and after,
    row counts, tables of the pages in use and the free list."""
    before, new = _geometry(case, seed)
    nseq = len(before)
    have = [_pages(b) for b in before]
    need = [_pages(b + t) - h for b, t, h in zip(before, new, have)]
    width = _pages(case["longest"] + case["tokens"]) + 3
    total = sum(have) + sum(need) + _FREE_SPARE
    order = torch.randperm(total, generator=torch.Generator().manual_seed(int(seed) * 31 + 3)).to(torch.int32)
    tables = torch.full((nseq, width), -1, dtype=torch.int32)
    at = 0
    for s, h in enumerate(have):
        tables[s, :h] = order[at:at + h]
        at += h
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return {"nseq": nseq, "rows": sum(new), "max_rows": max(new), "n_pages": total, "width": width, "before": before,
            "new": new, "lens": ints(before), "counts": ints(new), "tables": tables.cuda(), "free": order[at:].cuda(),
            "taken": ints([0])}


def _filled(case: dict, seed: int) -> dict:
    """Step inputs after the bookkeeping: every position's slot (page * 16 + place),
    sequence after sequence, and the new rows' among them."""
    t = _step_inputs(case, seed)
    tables, at, free = t["tables"].cpu(), 0, t["free"].cpu()
    slots, rows = [], []
    for s, (b, n) in enumerate(zip(t["before"], t["new"])):
        h, m = _pages(b), _pages(b + n)
        tables[s, h:m] = free[at:at + m - h]
        at += m - h
        p = torch.arange(b + n)
        slots.append(tables[s].long()[p // BLOCK] * BLOCK + p % BLOCK)
        rows.append(slots[-1][b:])
    t["tables"] = tables.cuda()
    t["old_slots"] = torch.cat([s[:b] for s, b in zip(slots, t["before"])]).to(torch.int32).cuda()
    t["slots"] = torch.cat(rows).to(torch.int32).cuda()
    ends = torch.tensor([0] + t["new"]).cumsum(0)
    t["row_start"] = ends.to(torch.int32).cuda()
    t["lens"] = t["lens"] + t["counts"]
    t["max_pages"] = max(_pages(b + n) for b, n in zip(t["before"], t["new"]))
    return t


def _kv_rows(case: dict, seed: int, n: int, stream: int):
    """K and V of n positions, [n, kv_heads * head_dim], in the case's type."""
    width, dtype = case["kv_heads"] * case["head_dim"], _TYPES[case["type"]]
    size = torch.exp(0.5 * _normal((width,), seed, 10))
    size[torch.randperm(width, generator=_gen(seed, 11), device="cuda")[:width // 64]] *= 4.0
    k = _normal((n, width), seed, stream)
    k *= size
    return k.to(dtype), _normal((n, width), seed, stream + 1).to(dtype)


def _inputs(case: dict, seed: int) -> dict:
    if case["kind"] == "tables":
        return _step_inputs(case, seed)
    t = _filled(case, seed)
    t["k_old"], t["v_old"] = _kv_rows(case, seed, t["old_slots"].numel(), 20)
    t["k"], t["v"] = _kv_rows(case, seed, t["rows"], 30)
    if case["kind"] == "write":
        # what is read back: all positions of the pages that the rows go to
        last = [(b // BLOCK * BLOCK, b, b + n) for b, n in zip(t["before"], t["new"])]
        old = []
        base = 0
        for lo, b, _ in last:
            old.append(t["old_slots"][base + lo:base + b])
            base += b
        t["read"] = torch.cat(old + [t["slots"]])
        return t
    shape = (t["rows"], case["heads"] * case["head_dim"])
    dtype = _TYPES[case["type"]]
    t["q"] = _normal(shape, seed, 40).to(dtype)
    t["gate"] = _normal(shape, seed, 41).to(dtype) if case["gate"] else None
    return t


# ---- plain form ---------------------------------------------------------------


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in f32 for whole e in [-126, 127], from its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _code_values(device) -> torch.Tensor:
    """Magnitudes of the e4m3 codes 0..126."""
    c = torch.arange(127, device=device)
    e, m = c // 8, (c % 8).float()
    return torch.where(e == 0, m / 512.0, (1.0 + m / 8.0) * _pow2(e - 7))


def _holds(top: torch.Tensor) -> torch.Tensor:
    """The smallest exponent e >= -126 with top <= 448 * 2^e (448 = 0.875 * 2^9)."""
    m, e = torch.frexp(top)
    e = e - 9 + (m > 0.875)
    return torch.where(top > 0, e, torch.full_like(e, -126)).clamp_min(-126)


def _to_codes(x: torch.Tensor) -> torch.Tensor:
    """f32 magnitudes up to 448 to e4m3 codes, to nearest, ties to the even code."""
    _, e = torch.frexp(x.abs())
    step = (e - 4).clamp_min(-9)
    near = torch.round(x.abs() * _pow2(-step)) * _pow2(step)
    return (torch.searchsorted(_code_values(x.device), near) + 128 * (x < 0)).to(torch.uint8)


class _Pages:
    """Codes u8 [pages, kv_heads, 16, head_dim] and exponents of K and V, and which
    positions are filled."""

    def __init__(self, case: dict, n_pages: int):
        self.kv, self.hd = case["kv_heads"], case["head_dim"]
        shape = (2, n_pages, self.kv, BLOCK, self.hd)
        self.codes = torch.zeros(shape, dtype=torch.uint8, device="cuda")
        self.exps = torch.full(shape[:3], -126, dtype=torch.int32, device="cuda")
        self.signed = torch.cat([v := _code_values("cuda"), v.new_zeros(1), -v, v.new_zeros(1)])

    def write(self, which: int, x: torch.Tensor, slots: torch.Tensor) -> None:
        """Rows x [n, kv * hd] into positions of K (0) or V (1); earlier positions of their pages stay."""
        slots = slots.long()
        pages, at = torch.unique(slots // BLOCK, return_inverse=True)
        new = torch.zeros((pages.numel(), BLOCK, self.kv, self.hd), device="cuda")
        new[at, slots % BLOCK] = x.float().reshape(-1, self.kv, self.hd)
        new = new.transpose(1, 2)
        here = torch.zeros((pages.numel(), BLOCK), dtype=torch.bool, device="cuda")
        here[at, slots % BLOCK] = True
        old_e = torch.where(here[:, :1], -126, self.exps[which, pages])  # a page written from its first place is new
        e = torch.maximum(old_e, _holds(new.abs().amax((2, 3))))
        old = self.signed[self.codes[which, pages].int()] * _pow2((old_e - e).clamp_min(-126))[..., None, None]
        units = torch.where(here[:, None, :, None], new * _pow2(-e)[..., None, None], old)
        first = here.int().argmax(1)
        past = torch.arange(BLOCK, device="cuda")[None] < first[:, None]
        units = units * (past | here)[:, None, :, None]
        self.codes[which, pages] = _to_codes(units)
        self.exps[which, pages] = e

    def values(self, which: int, pages: torch.Tensor) -> torch.Tensor:
        """f32 [pages, kv, 16, hd]"""
        pages = pages.long()
        return self.signed[self.codes[which, pages].int()] * _pow2(self.exps[which, pages])[..., None, None]

    def positions(self, which: int, pages: torch.Tensor, n: int) -> torch.Tensor:
        """f32 [kv, n, hd]: a sequence's first n positions"""
        return self.values(which, pages).transpose(0, 1).reshape(self.kv, -1, self.hd)[:, :n]


def _bounds(store: _Pages, pages: torch.Tensor, n: int) -> torch.Tensor:
    """[pages, kv, 2, hd]: highest and lowest key codes over a sequence's first n positions, in steps of 4, outward."""
    units = store.signed[store.codes[0, pages.long()].int()]
    filled = (torch.arange(pages.numel() * BLOCK, device="cuda") < n).reshape(-1, 1, BLOCK, 1)
    hi = torch.where(filled, units, -1e9).amax(2)
    lo = torch.where(filled, units, 1e9).amin(2)
    return torch.stack([torch.ceil(hi / 4), torch.floor(lo / 4)], 2)


class _Plain:
    def __init__(self, case: dict, seed: int):
        self.case, self.t = case, _inputs(case, seed)
        t = self.t
        if case["kind"] == "tables":
            return
        self.store = _Pages(case, t["n_pages"])
        if t["old_slots"].numel():
            self.store.write(0, t["k_old"], t["old_slots"])
            self.store.write(1, t["v_old"], t["old_slots"])
        if case["kind"] == "write":
            return
        self.store.write(0, t["k"], t["slots"])
        self.store.write(1, t["v"], t["slots"])
        for name in ("k_old", "v_old", "k", "v"):
            del t[name]
        self.ctx = [b + n for b, n in zip(t["before"], t["new"])]
        self.table = [t["tables"][s, :_pages(c)].long() for s, c in enumerate(self.ctx)]
        if case["kind"] == "sparse":
            self.bounds = [_bounds(self.store, p, c) for p, c in zip(self.table, self.ctx)]

    def run(self):
        return getattr(self, "_" + self.case["kind"])()

    def _tables(self):
        t = self.t
        lens, counts, tables = t["lens"].long(), t["counts"].long(), t["tables"].clone()
        have, want = (lens + BLOCK - 1) // BLOCK, (lens + counts + BLOCK - 1) // BLOCK
        ends = torch.cumsum(counts, 0)
        row_start = torch.cat([ends.new_zeros(1), ends])
        need = torch.cumsum(want - have, 0)
        seq = torch.repeat_interleave(torch.arange(t["nseq"], device="cuda"), counts)
        pos = torch.arange(t["rows"], device="cuda") - row_start[seq] + lens[seq]
        place = torch.repeat_interleave(torch.arange(t["nseq"], device="cuda"), want - have)
        first = need - (want - have)
        k = torch.arange(place.numel(), device="cuda")
        tables[place, have[place] + k - first[place]] = t["free"][t["taken"].long() + k]
        slots = tables[seq, pos // BLOCK].long() * BLOCK + pos % BLOCK
        i32 = lambda v: v.to(torch.int32)
        return [tables, i32(lens + counts), i32(t["taken"] + place.numel()), i32(row_start), i32(seq), i32(pos),
                i32(slots), torch.zeros_like(t["lens"])]

    def _write(self):
        t, st, out = self.t, self.store, []
        for which, x in ((0, t["k"]), (1, t["v"])):
            st.write(which, x, t["slots"])
            read = t["read"].long()
            units = st.signed[st.codes[which, read // BLOCK, :, read % BLOCK].int()]
            out.append((units * _pow2(st.exps[which, read // BLOCK])[..., None]).reshape(read.numel(), -1))
        return out

    def _finish(self, out):
        """[rows, heads * hd] f32 -> gate, type"""
        if self.t["gate"] is not None:
            out = out / (1.0 + torch.exp(-self.t["gate"].float()))
        return out.to(_TYPES[self.case["type"]])

    def _attn(self):
        c, t, out, at = self.case, self.t, [], 0
        kv, hd = c["kv_heads"], c["head_dim"]
        g = c["heads"] // kv
        for s, (n, ctx) in enumerate(zip(t["new"], self.ctx)):
            q = t["q"][at:at + n].float().reshape(n, kv, g, hd).permute(1, 2, 0, 3).reshape(kv, g * n, hd)
            k, v = (self.store.positions(i, self.table[s], ctx) for i in (0, 1))
            p = torch.matmul(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(hd))
            if n > 1:
                late = torch.arange(ctx, device="cuda")[None] > torch.arange(ctx - n, ctx, device="cuda")[:, None]
                p = p.reshape(kv, g, n, ctx).masked_fill(late, -math.inf).reshape(kv, g * n, ctx)
            p = torch.exp(p - p.amax(-1, keepdim=True))
            o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
            out.append(o.reshape(kv, g, n, hd).permute(2, 0, 1, 3).reshape(n, -1))
            at += n
        return self._finish(torch.cat(out))

    def _sparse(self):
        c, t, out, at = self.case, self.t, [], 0
        kv, hd, top = c["kv_heads"], c["head_dim"], c["top"]
        g = c["heads"] // kv
        sel = torch.full((t["rows"], kv, top), -1, dtype=torch.int32, device="cuda")
        count = torch.zeros((t["rows"], kv), dtype=torch.int32, device="cuda")
        for s, (n, ctx) in enumerate(zip(t["new"], self.ctx)):
            hi, lo = self.bounds[s].unbind(2)
            scale = _pow2(self.store.exps[0, self.table[s]])
            k, v = (self.store.values(i, self.table[s]) for i in (0, 1))
            for j in range(n):
                pos = ctx - n + j
                pages = pos // BLOCK + 1
                q = t["q"][at].float().reshape(kv, g, hd)
                m, e = torch.frexp(q.abs().amax((1, 2)))
                e = e - 7 + (m > 127 / 128)  # 127 * 2^e holds the largest
                q8 = torch.round(q * _pow2(-e)[:, None, None])
                score = (torch.matmul(q8.clamp_min(0), hi[:pages].permute(1, 2, 0).contiguous())
                         + torch.matmul(q8.clamp_max(0), lo[:pages].permute(1, 2, 0).contiguous())).amax(1)
                score = score * scale[:pages].t()
                score[:, :c["sinks"]] = math.inf
                score[:, max(pages - c["recent"], 0):] = math.inf
                m = min(top, pages)
                best = torch.sort(torch.sort(score, dim=1, descending=True, stable=True)[1][:, :m], dim=1)[0]
                sel[at, :, :m] = best.to(torch.int32)
                count[at] = m
                head = torch.arange(kv, device="cuda")[:, None]
                ks, vs = (x[best, head].reshape(kv, m * BLOCK, hd) for x in (k, v))
                p = torch.matmul(q, ks.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(hd))
                where = (best[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")).reshape(kv, 1, -1)
                p = p.masked_fill(where > pos, -math.inf)
                p = torch.exp(p - p.amax(-1, keepdim=True))
                out.append((torch.matmul(p, vs) / p.sum(-1, keepdim=True)).reshape(1, -1))
                at += 1
        return [self._finish(torch.cat(out)), sel, count]


# ---- the framework's calls ------------------------------------------------------

_dev = None


def _device():
    """The program's one device handle."""
    global _dev
    if _dev is None:
        from pagoda_amd import Device

        _dev = Device("hip")
    return _dev


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


class _Own:
    def __init__(self, case: dict, seed: int):
        from pagoda_amd.kv8 import Kv8Pool

        self.case, dev = case, _device()
        self.t = t = _inputs(case, seed)
        ints = lambda *shape: torch.empty(shape, dtype=torch.int32, device="cuda")
        if case["kind"] == "tables":
            n, rows = t["nseq"], t["rows"]
            self.out = [t["tables"], ints(n), ints(1), ints(n + 1), ints(rows), ints(rows), ints(rows), ints(n)]
            torch.cuda.synchronize()
            return
        self.kind = _TYPE_IDS[case["type"]]
        self.width = width = case["kv_heads"] * case["head_dim"]
        self.pool = Kv8Pool(dev, case["kv_heads"], case["head_dim"], t["n_pages"])
        torch.cuda.synchronize()  # the rows come from torch's stream, the device's reads them
        if t["old_slots"].numel():
            self.pool.append_dev(_ptr(t["k_old"]), width, _ptr(t["v_old"]), width, self.kind, _ptr(t["old_slots"]),
                                 t["old_slots"].numel())
        if case["kind"] == "write":
            n = t["read"].numel()
            self.out = [torch.empty((n, width), device="cuda") for _ in range(2)]
        else:
            self.pool.append_dev(_ptr(t["k"]), width, _ptr(t["v"]), width, self.kind, _ptr(t["slots"]), t["rows"])
            self.out = torch.empty_like(t["q"])
            self.args = (case["heads"], _ptr(t["q"]), t["q"].shape[1], self.kind, t["nseq"], _ptr(t["row_start"]),
                         _ptr(t["lens"]), _ptr(t["tables"]), t["width"], t["rows"])
            top = case.get("top", 0)
            size = (self.pool.sparse_ws_bytes(case["heads"], t["rows"], t["width"], top) if top else
                    self.pool.attn_ws_bytes(case["heads"], t["nseq"], t["width"], t["rows"]))
            self.ws = torch.empty((max(size, 16),), dtype=torch.uint8, device="cuda")
            self.gate = (_ptr(t["gate"]), t["q"].shape[1])
            if top:
                self.sel, self.count = ints(t["rows"], case["kv_heads"], top), ints(t["rows"], case["kv_heads"])
        dev.sync()  # the pages are written before the rows that they came from go
        for name in ("k_old", "v_old") + (() if case["kind"] == "write" else ("k", "v")):
            del t[name]

    def run(self):
        from pagoda_amd.kv8 import kv_tables_dev

        c, t = self.case, self.t
        kind, out = c["kind"], self.out
        if kind == "tables":
            kv_tables_dev(_device(), BLOCK, t["nseq"], _ptr(t["lens"]), _ptr(t["counts"]), _ptr(out[0]), t["width"],
                          _ptr(t["free"]), t["free"].numel(), _ptr(t["taken"]), t["rows"], *map(_ptr, out[1:]))
            return out
        if kind == "write":
            self.pool.append_dev(_ptr(t["k"]), self.width, _ptr(t["v"]), self.width, self.kind, _ptr(t["slots"]),
                                 t["rows"])
            self.pool.read_dev(_ptr(t["read"]), t["read"].numel(), _ptr(out[0]), self.width, _ptr(out[1]), self.width)
            return out
        if kind == "attn":
            self.pool.attn_dev(*self.args, t["max_rows"], _ptr(out), out.shape[1], _ptr(self.ws), self.ws.numel(),
                               *self.gate)
            return out
        self.pool.select_dev(*self.args, c["top"], c["sinks"], c["recent"], _ptr(self.sel), _ptr(self.count),
                             _ptr(self.ws), self.ws.numel())
        self.pool.attn_sparse_dev(*self.args, c["top"], _ptr(self.sel), _ptr(self.count), _ptr(out), out.shape[1],
                                  _ptr(self.ws), self.ws.numel(), *self.gate)
        return [out, self.sel, self.count]


def prepare(case: dict, seed: int):
    state = (_Own if own else _Plain)(case, seed)
    torch.cuda.synchronize()
    return state


def run(state):
    return state.run()


# ---- what a pass cannot do without ------------------------------------------------


def work(case: dict) -> dict:
    before, new = _geometry(case, 0)
    rows, kind = sum(new), case["kind"]
    if kind == "tables":
        fresh = sum(_pages(b + n) - _pages(b) for b, n in zip(before, new))
        return {"bytes": 4.0 * (2 * len(before) + 2 * fresh + 3 * len(before) + 3 * rows), "flops": 0.0}
    size, kv, hd = _TYPES[case["type"]].itemsize, case["kv_heads"], case["head_dim"]
    if kind == "write":
        old = sum(b % BLOCK for b in before)
        return {"bytes": 2.0 * kv * hd * (rows * (size + 1) + 2 * old + (rows + old) * 5), "flops": 4.0 * rows * kv * hd}
    heads = case["heads"]
    io = rows * heads * hd * size * (3 if case["gate"] else 2)
    if kind == "attn":
        attended = sum(n * b + n * (n + 1) // 2 for b, n in zip(before, new))
        return {"bytes": 2.0 * kv * hd * sum(b + n for b, n in zip(before, new)) + io, "flops": 4.0 * hd * heads * attended}
    pages = sum(_pages(b + n) for b, n in zip(before, new))
    read = sum(min(case["top"], _pages(b + j + 1)) for b, n in zip(before, new) for j in range(n))
    scored = sum(_pages(b + j + 1) for b, n in zip(before, new) for j in range(n))
    # (every row's own pages: rows of one sequence choose for themselves)
    return {"bytes": 2.0 * kv * hd * (pages + read * BLOCK) + io + 4.0 * rows * kv * (case["top"] + 1),
            "flops": 4.0 * hd * heads * read * BLOCK + 2.0 * hd * heads * scored}


# ---- the same values in 64 bits -----------------------------------------------------


def _exact_pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in float64 for whole e, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_round(x: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """float64 values to the nearest e4m3 multiple of 2^e, halves to even."""
    unit = x * _exact_pow2(-e)
    _, binade = torch.frexp(unit.abs().clamp_min(2.0 ** -6))
    step = _exact_pow2(binade - 4)
    return (unit / step).round() * step * _exact_pow2(e)


def _exact_exponent(x: torch.Tensor) -> torch.Tensor:
    """Over the positions and channels of [kv, positions, hd]: the exponent that holds the largest magnitude."""
    m, e = torch.frexp(x.abs().amax((1, 2)) / 448.0)
    return (e - (m == 0.5).int()).clamp_min(-126).double()[:, None, None]


def _exact_sequence(case: dict, t: dict, s: int, which: str):
    """A sequence's cached values [kv, ctx, hd] and their pages' exponents [kv, pages],
    page by page: what was there, then the step's rows."""
    kv, hd = case["kv_heads"], case["head_dim"]
    b, n = t["before"][s], t["new"][s]
    o, r = sum(t["before"][:s]), sum(t["new"][:s])
    rows = lambda x, i, m: x[i:i + m].double().reshape(m, kv, hd).transpose(0, 1)
    old, new = rows(t[which + "_old"], o, b), rows(t[which], r, n)

    def whole(x):  # full pages, and a last one, written at once: [kv, pages, 16, hd] -> values, exponents
        m = x.shape[1]
        pad = torch.cat([x, x.new_zeros((kv, -m % BLOCK, hd))], 1).reshape(kv, -1, BLOCK, hd)
        f, e = torch.frexp(pad.abs().amax((2, 3)) / 448.0)
        e = (e - (f == 0.5).int()).clamp_min(-126).double()
        e = torch.where(pad.abs().amax((2, 3)) > 0, e, torch.full_like(e, -126.0))
        return _exact_round(pad, e[..., None, None]).reshape(kv, -1, hd)[:, :m], e

    part = min(-b % BLOCK, n)  # new rows that share the last old page
    v_old, e_old = whole(old)
    v_new, e_new = whole(new[:, part:])
    if part:
        e = torch.maximum(e_old[:, -1:, None], _exact_exponent(new[:, :part]))
        cut = b // BLOCK * BLOCK
        v_old = torch.cat([v_old[:, :cut], _exact_round(v_old[:, cut:], e), _exact_round(new[:, :part], e)], 1)
        e_old = torch.cat([e_old[:, :-1], e[:, :, 0]], 1)
    return torch.cat([v_old, v_new], 1), torch.cat([e_old, e_new], 1)


def _exact_tables(t: dict):
    taken, free = 0, t["free"].tolist()
    tables, seq, pos, slots, starts = t["tables"].tolist(), [], [], [], [0]
    for s, (b, n) in enumerate(zip(t["before"], t["new"])):
        for p in range(b, b + n):
            if p % BLOCK == 0:
                tables[s][p // BLOCK] = free[taken]
                taken += 1
            seq.append(s)
            pos.append(p)
            slots.append(tables[s][p // BLOCK] * BLOCK + p % BLOCK)
        starts.append(len(seq))
    lens = [b + n for b, n in zip(t["before"], t["new"])]
    return [torch.tensor(v, dtype=torch.int32) for v in (tables, lens, [taken], starts, seq, pos, slots, [0] * len(lens))]


def exact(case: dict, seed: int):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "tables":
        return _exact_tables(t)
    kv, hd = case["kv_heads"], case["head_dim"]
    if kind == "write":
        out = []
        for which in ("k", "v"):
            seqs = [_exact_sequence(case, t, s, which)[0].transpose(0, 1) for s in range(t["nseq"])]
            parts = [x[b // BLOCK * BLOCK:b] for x, b in zip(seqs, t["before"])] + [x[b:] for x, b in zip(seqs, t["before"])]
            out.append(torch.cat(parts).reshape(-1, kv * hd))
        return out
    g = case["heads"] // kv
    outs, sels, counts, at = [], [], [], 0
    for s, (b, n) in enumerate(zip(t["before"], t["new"])):
        k, e = _exact_sequence(case, t, s, "k")
        v, _ = _exact_sequence(case, t, s, "v")
        for r0 in range(0, n, 64):
            m = min(64, n - r0)
            q = t["q"][at + r0:at + r0 + m].double().reshape(m, kv, g, hd)
            x = torch.stack([q[:, h].reshape(m * g, hd) @ k[h].t().contiguous() for h in range(kv)]) / math.sqrt(hd)
            x = x.reshape(kv, m, g, b + n)
            seen = torch.arange(b + n, device="cuda")[None] <= torch.arange(b + r0, b + r0 + m, device="cuda")[:, None]
            seen = seen[None].expand(kv, m, b + n)
            if kind == "sparse":
                picked = _exact_pick(case, q, k, e, [b + r0 + j + 1 for j in range(m)])
                sels.append(picked[0])
                counts.append(picked[1])
                seen = seen & picked[2]
            w = torch.softmax(x.masked_fill(~seen[:, :, None], -math.inf), -1)
            o = torch.stack([w[h].reshape(m * g, b + n) @ v[h] for h in range(kv)], 1)
            outs.append(o.reshape(m, g, kv, hd).transpose(1, 2).reshape(m, -1))
        at += n
    out = torch.cat(outs)
    if t["gate"] is not None:
        out = out * torch.sigmoid(t["gate"].double())
    return out if kind == "attn" else [out, torch.cat(sels), torch.cat(counts)]


def _exact_pick(case: dict, q: torch.Tensor, k: torch.Tensor, e: torch.Tensor, lens: list[int]):
    """Selected pages [m, kv, top] (-1 behind them), their number, and the positions [kv, m, ctx] they hold."""
    kv, hd, top = case["kv_heads"], case["head_dim"], case["top"]
    ctx, pages = k.shape[1], e.shape[1]
    codes = k * _exact_pow2(-e.repeat_interleave(BLOCK, 1))[:, :ctx, None]
    fill = codes.new_zeros((kv, pages * BLOCK - ctx, hd))
    hi = torch.cat([codes, fill - math.inf], 1).reshape(kv, pages, BLOCK, hd).amax(2).div(4).ceil()
    lo = torch.cat([codes, fill + math.inf], 1).reshape(kv, pages, BLOCK, hd).amin(2).div(4).floor()
    sel = torch.full((len(lens), kv, top), -1, dtype=torch.int32)
    count = torch.zeros((len(lens), kv), dtype=torch.int32)
    seen = torch.zeros((kv, len(lens), pages * BLOCK), dtype=torch.bool, device="cuda")
    for j, n in enumerate(lens):
        here = _pages(n)
        for h in range(kv):
            best = torch.full((here,), -math.inf, dtype=torch.float64, device="cuda")
            largest = float(q[j, h].abs().max())
            step = 2.0 ** math.ceil(math.log2(largest / 127)) if largest else 1.0
            if largest / step > 127:  # (the logarithm's own rounding)
                step *= 2
            for row in torch.round(q[j, h] / step):
                best = torch.maximum(best, torch.where(row > 0, row * hi[h, :here], row * lo[h, :here]).sum(1))
            rank = (best * _exact_pow2(e[h, :here])).tolist()
            forced = set(range(min(case["sinks"], here))) | set(range(max(here - case["recent"], 0), here))
            order = sorted(range(here), key=lambda p: (p not in forced, -rank[p], p))[:top]
            order.sort()
            sel[j, h, :len(order)] = torch.tensor(order, dtype=torch.int32)
            count[j, h] = len(order)
            seen.view(kv, len(lens), pages, BLOCK)[h, j, torch.tensor(order, device="cuda")] = True
    return sel, count, seen[:, :, :ctx]
