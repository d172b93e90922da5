"""Timed cases of the MXFP4 operators: microscaled 4-bit weights and activations.

An MXFP4 block is 32 consecutive elements of a row: 4-bit floating-point codes
(sign, 0 .5 1 1.5 2 3 4 6; element 2i in the low nibble of byte i) and one
scale byte s that stands for 2^(s - 127). Kinds of case (`kind`):

  quant   rows of f32, f16 or bf16 to MXFP4 and the values that the codes stand
          for: what runs before a product of two MXFP4 operands, and over the
          weights when a matrix is quantized on the device.
  lin     one projection with MXFP4 weights, activations as they are (f32, f16
          or bf16), with or without the residual: a decode step's rows, or a
          prompt's.
  glu     the gate / up pair of a feed-forward block in that form:
          silu(gate x) * (up x).
  mx      one projection of MXFP4 rows with MXFP4 weights.
  glumx   the gate / up pair of MXFP4 rows.

Weights are N(0, 0.02) quantized to MXFP4. Activation rows are of unit
variance, as an RMSNorm leaves them, with a few channels twenty times as large.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 2}
_LARGEST = 4096 * 5120 * 17408  # products of the largest listed case


def listed() -> list[dict]:
    return [
        # one decode row before a projection: the smallest call
        {"name": "quant_1", "kind": "quant", "rows": 1, "k": 896, "type": "bf16"},
        # a prompt's feed-forward rows before the down projection
        {"name": "quant_2048", "kind": "quant", "rows": 2048, "k": 17408, "type": "f32"},
        # the 0.5B model's q|k|v projection of one decode row
        {"name": "lin_1", "kind": "lin", "rows": 1, "n": 1152, "k": 896, "type": "f32", "res": False},
        # its lm_head for a few requests
        {"name": "lin_head_5", "kind": "lin", "rows": 5, "n": 151936, "k": 896, "type": "f16", "res": False},
        # the 27B-class down projection of a served batch, with the residual
        {"name": "lin_32", "kind": "lin", "rows": 32, "n": 5120, "k": 17408, "type": "bf16", "res": True},
        # a projection over an odd number of a prompt's rows
        {"name": "lin_1999", "kind": "lin", "rows": 1999, "n": 5120, "k": 6144, "type": "bf16", "res": False},
        # the 27B-class gate / up pair: one user, and a short prompt
        {"name": "glu_1", "kind": "glu", "rows": 1, "n": 17408, "k": 5120, "type": "f32"},
        {"name": "glu_333", "kind": "glu", "rows": 333, "n": 17408, "k": 5120, "type": "f32"},
        # MXFP4 rows: a small batch through the down projection, a long prompt through one gate / up matrix
        {"name": "mx_8", "kind": "mx", "rows": 8, "n": 5120, "k": 17408, "res": True},
        {"name": "mx_4096", "kind": "mx", "rows": 4096, "n": 17408, "k": 5120, "res": False},
        # the pair: a served batch, and a prompt chunk
        {"name": "glumx_48", "kind": "glumx", "rows": 48, "n": 17408, "k": 5120},
        {"name": "glumx_2048", "kind": "glumx", "rows": 2048, "n": 17408, "k": 5120},
    ]


def _log(rng, lo: int, hi: int, step: int = 1) -> int:
    """A multiple of step, spread over the logarithm of [lo, hi]."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng) -> dict:
    kind = rng.choice(["quant", "lin", "lin", "glu", "mx", "mx", "glumx"])
    if kind == "quant":
        k = _log(rng, 64, 17408, 32)
        return {"kind": kind, "rows": _log(rng, 1, 2048), "k": k, "type": rng.choice(sorted(_TYPES))}
    pair = 2 if kind in ("glu", "glumx") else 1
    k = _log(rng, 64, 17408, 32)
    n = _log(rng, 100, 151936 // pair)
    n = min(n, 17408 * 5120 * 2 // (pair * k))
    rows = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 64, 4096)
    rows = max(1, min(rows, _LARGEST // (pair * n * k * (2 if kind in ("lin", "glu") else 1)), 4096 * 17408 // n))
    case = {"kind": kind, "rows": rows, "n": n, "k": k}
    if kind == "lin":
        case["type"] = rng.choice(sorted(_TYPES))
    if kind == "glu":
        case["type"] = "f32"
    if kind in ("lin", "mx"):
        case["res"] = rng.random() < 0.5
    return case


# ---- inputs -------------------------------------------------------------------


def _gen(seed: int, stream: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1_000_003 + stream) & 0x7FFFFFFFFFFFFFFF)
    return g


def _normal(shape, seed: int, stream: int, scale: float = 1.0) -> torch.Tensor:
    return torch.randn(shape, generator=_gen(seed, stream), device="cuda") * scale


def _rows_in(case: dict, seed: int) -> torch.Tensor:
    """Activation rows [rows, k] in f32."""
    k = case["k"]
    x = _normal((case["rows"], k), seed, 1)
    far = torch.randperm(k, generator=_gen(seed, 2), device="cuda")[:max(1, k // 256)]
    x[:, far] *= 20.0
    return x


def _pad16(v: int) -> int:
    return (v + 15) // 16 * 16


def _pack(x: torch.Tensor):
    """Rows of f32 as MXFP4 planes: codes u8 [rows, k / 2] and scales u8 [rows,
    k / 32 padded to a multiple of 16]."""
    rows, k = x.shape
    b = x.reshape(rows, k // 32, 32)
    _, e = torch.frexp(b.abs().amax(-1))  # max = m * 2^e, m in [0.5, 1)
    s = (e + 124).clamp(0, 254)
    u = torch.ldexp(b, 127 - s[..., None])
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    a = u.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i, edge in enumerate(edges):  # a tie goes to the even code
        code += (a > edge) if i % 2 == 0 else (a >= edge)
    code |= (b < 0).to(torch.uint8) << 3
    code = code.reshape(rows, k)
    scales = torch.zeros((rows, _pad16(k // 32)), dtype=torch.uint8, device=x.device)
    scales[:, :k // 32] = s.to(torch.uint8)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), scales


def _weights(case: dict, seed: int, stream: int):
    return _pack(_normal((case["n"], case["k"]), seed, stream, 0.02))


def _inputs(case: dict, seed: int) -> dict:
    kind = case["kind"]
    t = {"x": _rows_in(case, seed)}
    if kind in ("quant", "lin", "glu"):
        t["x"] = t["x"].to(_TYPES[case["type"]])
    else:
        t["x"] = _pack(t["x"])
    if kind != "quant":
        t["w"] = _weights(case, seed, 3)
    if kind in ("glu", "glumx"):
        t["up"] = _weights(case, seed, 4)
    if case.get("res"):
        t["res"] = _normal((case["rows"], case["n"]), seed, 5)
    return t


# ---- plain form ---------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _values(planes) -> torch.Tensor:
    """The f32 values [rows, k] that MXFP4 planes stand for."""
    codes, scales = planes
    rows, half = codes.shape
    table = torch.tensor(_E2M1, device=codes.device)
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).reshape(rows, -1, 32)
    step = torch.exp2(scales[:, :half // 16].float() - 127.0)
    return (v * step[..., None]).reshape(rows, 2 * half)


class _Plain:
    def __init__(self, case: dict, seed: int):
        self.case, self.t = case, _inputs(case, seed)

    def run(self):
        kind, t = self.case["kind"], self.t
        if kind == "quant":
            return _values(_pack(t["x"].float()))
        x = t["x"].float() if kind in ("lin", "glu") else _values(t["x"])
        y = x @ _values(t["w"]).t()
        if "up" in t:
            y = y / (1.0 + torch.exp(-y)) * (x @ _values(t["up"]).t())
        if "res" in t:
            y = t["res"] + y
        return y


# ---- the framework's calls ------------------------------------------------------

_dev = None


def _device():
    """The program's one device handle."""
    global _dev
    if _dev is None:
        from pagoda_amd import Device

        _dev = Device("hip")
    return _dev


def _matrix(planes):
    from pagoda_amd import Matrix

    codes, scales = planes
    return Matrix.from_mxfp4_dev(_device(), codes.data_ptr(), codes.stride(0), scales.data_ptr(), scales.stride(0),
                                 codes.shape[0], 2 * codes.shape[1])


class _Own:
    def __init__(self, case: dict, seed: int):
        self.case, dev = case, _device()
        t = _inputs(case, seed)
        torch.cuda.synchronize()  # the planes come from torch's stream, the handles are made on the device's
        self.x, self.res = t["x"], t.get("res")
        self.w = _matrix(t["w"]) if "w" in t else None
        self.up = _matrix(t["up"]) if "up" in t else None
        rows, k = case["rows"], case["k"]
        self.y = torch.empty((rows, case.get("n", k)), device="cuda")
        if case["kind"] == "quant":
            self.codes = torch.empty((rows, _pad16(k // 2)), dtype=torch.uint8, device="cuda")
            self.scales = torch.empty((rows, _pad16(k // 32)), dtype=torch.uint8, device="cuda")
        dev.sync()  # the handles are complete before the planes they came from go

    def run(self):
        from pagoda_amd import Matrix
        from pagoda_amd.matrix import mxfp4_quantize_dev

        c, y, rows, k = self.case, self.y, self.case["rows"], self.case["k"]
        kind = c["kind"]
        res = self.res.data_ptr() if self.res is not None else 0
        if kind == "quant":
            mxfp4_quantize_dev(_device(), self.x.data_ptr(), _TYPE_IDS[c["type"]], k, rows, k, self.codes.data_ptr(),
                               self.codes.stride(0), self.scales.data_ptr(), self.scales.stride(0), y.data_ptr(), k)
        elif kind == "lin":
            self.w.gemv_dev(self.x.data_ptr(), k, rows, y.data_ptr(), c["n"], _TYPE_IDS[c["type"]], res, c["n"])
        elif kind == "glu":
            Matrix.gemv_swiglu_dev(self.w, self.up, self.x.data_ptr(), k, rows, y.data_ptr(), c["n"])
        else:
            codes, scales = self.x
            planes = (codes.data_ptr(), codes.stride(0), scales.data_ptr(), scales.stride(0))
            if kind == "mx":
                self.w.gemv_mx_dev(*planes, rows, y.data_ptr(), c["n"], res, c["n"])
            else:
                Matrix.gemv_swiglu_mx_dev(self.w, self.up, *planes, rows, y.data_ptr(), c["n"])
        return y


def prepare(case: dict, seed: int):
    state = (_Own if own else _Plain)(case, seed)
    torch.cuda.synchronize()
    return state


def run(state):
    return state.run()


# ---- what a pass cannot do without ------------------------------------------------


def work(case: dict) -> dict:
    kind, rows, k = case["kind"], case["rows"], case["k"]
    size = _TYPES[case["type"]].itemsize if "type" in case else 17 / 32
    if kind == "quant":
        return {"bytes": rows * k * (size + 17 / 32 + 4), "flops": 6.0 * rows * k}
    n, pair = case["n"], 2 if kind in ("glu", "glumx") else 1
    return {"bytes": pair * n * k * 17 / 32 + rows * k * size + rows * n * 4 * (2 if case.get("res") else 1),
            "flops": 2.0 * pair * rows * n * k}


# ---- the same values in 64 bits -----------------------------------------------------


def _exact_values(planes) -> torch.Tensor:
    """float64 values of MXFP4 planes from the codes' fields: sign, two exponent
    bits and one mantissa bit (no implicit one where the exponent is 0)."""
    codes, scales = planes
    rows, half = codes.shape
    out = torch.empty((rows, half, 2), dtype=torch.float64, device=codes.device)
    for i in range(2):
        c = (codes >> (4 * i)) & 15
        e, m = ((c >> 1) & 3).double(), (c & 1).double()
        mag = torch.where(e == 0, m * 0.5, (1.0 + 0.5 * m) * 2.0 ** (e - 1.0))
        out[..., i] = torch.where(c >= 8, -mag, mag)
    scale = 2.0 ** (scales[:, :half // 16].double() - 127.0)
    return (out.reshape(rows, -1, 32) * scale[..., None]).reshape(rows, 2 * half)


def _exact_round(x: torch.Tensor) -> torch.Tensor:
    """float64 rows rounded to the values of their MXFP4 form: a multiple of the
    step of the value's binade, halves to even, at most 6 block scales."""
    b = x.reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    scale = 2.0 ** (torch.floor(torch.log2(top.clamp_min(2.0 ** -126))) - 2.0).clamp_min(-127.0)
    v = b / scale
    step = 2.0 ** (torch.floor(torch.log2(v.abs().clamp_min(1.0))) - 1.0)
    return (((v / step).round() * step).clamp(-6.0, 6.0) * scale).reshape(x.shape)


def exact(case: dict, seed: int):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "quant":
        return _exact_round(t["x"].double())
    x = t["x"].double() if kind in ("lin", "glu") else _exact_values(t["x"])
    y = x @ _exact_values(t["w"]).t()
    if "up" in t:
        y = y * torch.sigmoid(y) * (x @ _exact_values(t["up"]).t())
    return t["res"].double() + y if "res" in t else y
