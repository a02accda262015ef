"""ctypes binding of the microscaled 4-bit operators (include/minicompiler_b200_device.h).

As in the rest of the device layer, operands are device addresses (ints, e.g. torch tensors' data_ptr()) that the caller
owns, calls act on the current device and are enqueued on `stream` (a cudaStream_t as an int; 0 = the legacy default
stream). Types are "f32", "bf16" and "f16", 4-bit formats "e8m0_32" and "e4m3_16". A program that repeats a product
keeps the Fp4Gemm object and calls its enqueue().
"""

from __future__ import annotations

import ctypes as C
from collections import namedtuple

from .api import McError, _device_error, lib

FORMATS = {"e8m0_32": 1, "e4m3_16": 2}
TYPES = {"f32": 0, "bf16": 1, "f16": 2}

Fp4Sizes = namedtuple("Fp4Sizes", "code_pitch codes_bytes scales_bytes")


class _Fp4Tensor(C.Structure):
    _fields_ = [("format", C.c_int), ("batch", C.c_int), ("rows", C.c_longlong), ("cols", C.c_longlong), ("codes", C.c_void_p),
                ("scales", C.c_void_p), ("tensor_scale", C.c_void_p)]


class _Fp4GemmArgs(C.Structure):
    _fields_ = [("a", _Fp4Tensor), ("b", _Fp4Tensor), ("c", C.c_void_p), ("c_type", C.c_int), ("ldc", C.c_longlong),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t), ("status", C.c_void_p)]


def _format(name: str) -> int:
    if name not in FORMATS:
        raise McError(f"unknown 4-bit format '{name}': {', '.join(FORMATS)}")
    return FORMATS[name]


def _type(name: str) -> int:
    if name not in TYPES:
        raise McError(f"unknown type '{name}': {', '.join(TYPES)}")
    return TYPES[name]


def _check(rc: int) -> None:
    if rc != 0:
        raise McError(_device_error())


class Fp4Matrix:
    """`batch` matrices [rows, cols] in a 4-bit format, in device memory at `codes` and `scales` (mcd_fp4_tensor)."""

    def __init__(self, fmt: str, rows: int, cols: int, codes: int, scales: int, tensor_scale: int = 0, batch: int = 1):
        self.format, self.rows, self.cols, self.batch = fmt, rows, cols, batch
        self._c = _Fp4Tensor(_format(fmt), batch, rows, cols, codes or None, scales or None, tensor_scale or None)
        self._ref = C.byref(self._c)


def fp4_sizes(fmt: str, rows: int, cols: int, batch: int = 1) -> Fp4Sizes:
    """Bytes per row of codes, and of the two arrays of `batch` matrices [rows, cols]."""
    L = lib()
    return Fp4Sizes(L.mcd_fp4_code_pitch(cols), L.mcd_fp4_codes_bytes(rows, cols, batch),
                    L.mcd_fp4_scales_bytes(_format(fmt), rows, cols, batch))


def fp4_tensor_scale(src: int, dtype: str, rows: int, cols: int, out: int, pitch: int = 0, batch: int = 1, stream: int = 0) -> None:
    """mcd_fp4_tensor_scale: the f32 scale of each of `batch` matrices, into `out`."""
    _check(lib().mcd_fp4_tensor_scale(_type(dtype), src, rows, cols, pitch or cols, batch, out, stream))


def fp4_quantize(src: int, dtype: str, dst: Fp4Matrix, pitch: int = 0, stream: int = 0) -> None:
    """mcd_fp4_quantize: [batch, rows, cols] values at `src` into `dst`."""
    _check(lib().mcd_fp4_quantize(_type(dtype), src, pitch or dst.cols, dst._ref, stream))


def fp4_dequantize(src: Fp4Matrix, dst: int, dtype: str, pitch: int = 0, stream: int = 0) -> None:
    """mcd_fp4_dequantize: the values `src` stands for, to `dst`."""
    _check(lib().mcd_fp4_dequantize(src._ref, _type(dtype), dst, pitch or src.cols, stream))


def fp4_gemm_workspace_bytes(fmt: str, m: int, n: int, k: int) -> int:
    args = _Fp4GemmArgs()
    args.a = _Fp4Tensor(_format(fmt), 1, m, k, None, None, None)
    args.b = _Fp4Tensor(_format(fmt), 1, n, k, None, None, None)
    return lib().mcd_fp4_gemm_workspace(C.byref(args))


class Fp4Gemm:
    """mcd_fp4_gemm: c[m, n] = a[m, k] * b[n, k]^T, kept for any number of enqueue() calls.

    `status`, a device word that is 0 at first, is where a kernel says that it gave up a wait of two seconds and left c
    unfinished. Without one that shows nowhere: a program that has to know gives a word and looks at it where it reads c."""

    def __init__(self, a: Fp4Matrix, b: Fp4Matrix, c: int, c_dtype: str, ldc: int = 0, workspace: int = 0, workspace_bytes: int = 0,
                 status: int = 0):
        self._args = _Fp4GemmArgs(a._c, b._c, c or None, _type(c_dtype), ldc or b.rows, workspace or None, workspace_bytes, status or None)
        self._ref = C.byref(self._args)
        self._call = lib().mcd_fp4_gemm

    def enqueue(self, stream: int = 0) -> None:
        _check(self._call(self._ref, stream))

    @property
    def launches(self) -> int:
        return lib().mcd_fp4_gemm_launches(self._ref)
