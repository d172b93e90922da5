"""Quantized matrix handle (QuantMatrix, pagoda-hf/src/qwen3_gemv.rs:640-760)."""
from __future__ import annotations

import ctypes as C
from operator import index

import numpy as np

from ._lib import call
from .device import Device

FMT_A8, FMT_Q4K, FMT_Q6K, FMT_Q8_0, FMT_Q5_0, FMT_MXFP4 = 0, 1, 2, 3, 4, 5
FMT_NAMES = {FMT_A8: "a8", FMT_Q4K: "q4k", FMT_Q6K: "q6k", FMT_Q8_0: "q8_0", FMT_Q5_0: "q5_0", FMT_MXFP4: "mxfp4"}
# activation rows of MXFP4 products and of mxfp4_quantize_dev
X_F32, X_F16, X_BF16 = 0, 1, 2


def _ptr(a: np.ndarray) -> C.c_void_p:
    return a.ctypes.data_as(C.c_void_p)


# Device addresses go to the library as index(p or 0): whole numbers, or None for none. (ctypes
# would also take bytes, strings and arrays, as the addresses of host memory.)


def act_bytes(nrows: int, k: int) -> int:
    from ._lib import lib

    return int(lib().pgd_act_bytes(nrows, k))


def act_prep_dev(dev: Device, x_ptr: int, ldx: int, nrows: int, k: int, act_ptr: int) -> None:
    call("pgd_act_prep_dev", dev.handle, C.c_void_p(x_ptr), ldx, nrows, k, C.c_void_p(act_ptr))


def mxfp4_quantize_dev(dev: Device, x_ptr: int, x_type: int, ldx: int, nrows: int, k: int, codes_ptr: int, ldc: int,
                       scales_ptr: int, lds: int, values_ptr: int = 0, ldv: int = 0) -> None:
    """Rows of f32 / f16 / bf16 (x_type) to MXFP4 planes; values_ptr also receives the values they stand for."""
    call("pgd_mxfp4_quantize_dev", dev.handle, index(x_ptr or 0), x_type, ldx, nrows, k, index(codes_ptr or 0), ldc,
         index(scales_ptr or 0), lds, index(values_ptr or 0), ldv)


class Matrix:
    def __init__(self, dev: Device, handle: C.c_void_p):
        self.dev = dev
        self.handle = handle
        fmt, n_out, n_in = C.c_int(), C.c_int(), C.c_int()
        dbytes, abytes = C.c_size_t(), C.c_double()
        call("pgd_matrix_info", handle, C.byref(fmt), C.byref(n_out), C.byref(n_in), C.byref(dbytes), C.byref(abytes))
        self.fmt, self.n_out, self.n_in = fmt.value, n_out.value, n_in.value
        self.dev_bytes, self.algo_bytes = dbytes.value, abytes.value

    # ---- constructors ----
    @classmethod
    def upload_a8(cls, dev: Device, packed: np.ndarray, scales: np.ndarray, biases: np.ndarray, n_out: int, n_in: int):
        packed = np.ascontiguousarray(packed, np.uint32)
        scales = np.ascontiguousarray(scales, np.uint16)
        biases = np.ascontiguousarray(biases, np.uint16)
        assert packed.size == n_out * n_in // 4 and scales.size == biases.size == n_out * (n_in // 64)
        h = C.c_void_p()
        call("pgd_matrix_upload_a8", dev.handle, _ptr(packed), _ptr(scales), _ptr(biases), n_out, n_in, C.byref(h))
        return cls(dev, h)

    @classmethod
    def upload_kq(cls, dev: Device, fmt: int, blocks: np.ndarray, n_out: int, n_in: int):
        """GGML blocks, row-major: Q4_K / Q6_K super-blocks or Q8_0 / Q5_0 blocks."""
        blocks = np.ascontiguousarray(blocks, np.uint8)
        if fmt in (FMT_Q8_0, FMT_Q5_0):
            assert blocks.size == n_out * (n_in // 32) * (34 if fmt == FMT_Q8_0 else 22)
        else:
            assert blocks.size == n_out * ((n_in + 255) // 256) * (144 if fmt == FMT_Q4K else 210)
        h = C.c_void_p()
        name = {FMT_Q4K: "pgd_matrix_upload_q4k", FMT_Q6K: "pgd_matrix_upload_q6k", FMT_Q8_0: "pgd_matrix_upload_q8_0",
                FMT_Q5_0: "pgd_matrix_upload_q5_0"}[fmt]
        call(name, dev.handle, _ptr(blocks), n_out, n_in, C.byref(h))
        return cls(dev, h)

    @classmethod
    def upload_mxfp4(cls, dev: Device, codes: np.ndarray, scales: np.ndarray, n_out: int, n_in: int):
        """MXFP4 planes, row-major: codes [n_out, n_in / 2], scales [n_out, n_in / 32]."""
        codes = np.ascontiguousarray(codes, np.uint8)
        scales = np.ascontiguousarray(scales, np.uint8)
        assert codes.size == n_out * (n_in // 2) and scales.size == n_out * (n_in // 32)
        h = C.c_void_p()
        call("pgd_matrix_upload_mxfp4", dev.handle, _ptr(codes), _ptr(scales), n_out, n_in, C.byref(h))
        return cls(dev, h)

    @classmethod
    def from_mxfp4_dev(cls, dev: Device, codes_ptr: int, ldc: int, scales_ptr: int, lds: int, n_out: int, n_in: int):
        """MXFP4 planes in device memory (queued: they may go once the handle's stream has passed)."""
        h = C.c_void_p()
        call("pgd_matrix_from_mxfp4_dev", dev.handle, C.c_void_p(codes_ptr), ldc, C.c_void_p(scales_ptr), lds, n_out,
             n_in, C.byref(h))
        return cls(dev, h)

    @classmethod
    def synth(cls, dev: Device, fmt: int, n_out: int, n_in: int, seed: int, key: int, std: float = 0.02):
        h = C.c_void_p()
        call("pgd_matrix_synth", dev.handle, fmt, n_out, n_in, C.c_uint64(seed), C.c_uint64(key), C.c_float(std), C.byref(h))
        return cls(dev, h)

    def free(self) -> None:
        if self.handle:
            call("pgd_matrix_free", self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    # ---- ops ----
    def dequant(self, row0: int = 0, rows: int | None = None) -> np.ndarray:
        rows = self.n_out - row0 if rows is None else rows
        out = np.empty((rows, self.n_in), np.float32)
        call("pgd_matrix_dequant", self.handle, row0, rows, _ptr(out))
        return out

    def gemv(self, x: np.ndarray) -> np.ndarray:
        x = np.ascontiguousarray(x, np.float32)
        squeeze = x.ndim == 1
        x2 = x.reshape(-1, self.n_in)
        y = np.empty((x2.shape[0], self.n_out), np.float32)
        call("pgd_matrix_gemv", self.handle, _ptr(x2), x2.shape[0], _ptr(y))
        return y[0] if squeeze else y

    def gemv_dev(self, x_ptr: int, ldx: int, nrows: int, y_ptr: int, ldy: int, x_f16: int = False,
                 res_ptr: int = 0, ldres: int = 0) -> None:
        """x_f16: f32 rows (False), f16 (True), or for MXFP4 matrices X_F32 / X_F16 / X_BF16."""
        call("pgd_matrix_gemv_dev", self.handle, index(x_ptr or 0), int(x_f16), ldx, nrows, index(y_ptr or 0), ldy,
             index(res_ptr or 0), ldres)

    def gemv_q8act_dev(self, x_ptr: int, ldx: int, nrows: int, y_ptr: int, ldy: int, res_ptr: int = 0,
                       ldres: int = 0) -> None:
        """candle's CPU quantized matmul arithmetic (activations quantized to Q8_K / Q8_0)."""
        call("pgd_matrix_gemv_q8act_dev", self.handle, C.c_void_p(x_ptr), ldx, nrows, C.c_void_p(y_ptr), ldy,
             C.c_void_p(res_ptr or None), ldres)

    def gemv_q8act_pair_dev(self, ya_ptr: int, other: "Matrix", yb_ptr: int, x_ptr: int, ldx: int, nrows: int,
                            ldy: int) -> None:
        """This matrix and `other` over the same rows in one launch (candle's CPU arithmetic)."""
        call("pgd_matrix_gemv_q8act_pair_dev", self.handle, C.c_void_p(ya_ptr), other.handle, C.c_void_p(yb_ptr),
             C.c_void_p(x_ptr), ldx, nrows, ldy)

    def gemv_act_dev(self, act_ptr: int, nrows: int, y_ptr: int, ldy: int, res_ptr: int = 0, ldres: int = 0) -> None:
        call("pgd_matrix_gemv_act_dev", self.handle, C.c_void_p(act_ptr), nrows, C.c_void_p(y_ptr), ldy,
             C.c_void_p(res_ptr or None), ldres)

    @staticmethod
    def gemv_swiglu_act_dev(gate: "Matrix", up: "Matrix", act_ptr: int, nrows: int, mid_ptr: int, ldm: int):
        call("pgd_matrix_gemv_swiglu_act_dev", gate.handle, up.handle, C.c_void_p(act_ptr), nrows, C.c_void_p(mid_ptr), ldm)

    @staticmethod
    def gemv_swiglu_dev(gate: "Matrix", up: "Matrix", x_ptr: int, ldx: int, nrows: int, mid_ptr: int, ldm: int):
        call("pgd_matrix_gemv_swiglu_dev", gate.handle, up.handle, index(x_ptr or 0), ldx, nrows, index(mid_ptr or 0), ldm)

    def gemv_mx_dev(self, codes_ptr: int, ldc: int, scales_ptr: int, lds: int, nrows: int, y_ptr: int, ldy: int,
                    res_ptr: int = 0, ldres: int = 0) -> None:
        """MXFP4 rows (planes) times this MXFP4 matrix."""
        call("pgd_matrix_gemv_mx_dev", self.handle, index(codes_ptr or 0), ldc, index(scales_ptr or 0), lds, nrows,
             index(y_ptr or 0), ldy, index(res_ptr or 0), ldres)

    @staticmethod
    def gemv_swiglu_mx_dev(gate: "Matrix", up: "Matrix", codes_ptr: int, ldc: int, scales_ptr: int, lds: int,
                           nrows: int, mid_ptr: int, ldm: int):
        call("pgd_matrix_gemv_swiglu_mx_dev", gate.handle, up.handle, index(codes_ptr or 0), ldc, index(scales_ptr or 0),
             lds, nrows, index(mid_ptr or 0), ldm)
