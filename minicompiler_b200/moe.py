"""ctypes binding of the mixture-of-experts layer (include/minicompiler_b200_device.h); conventions as in fp4.py."""

from __future__ import annotations

import ctypes as C

from .api import lib
from .fp4 import Fp4Matrix, _check, _Fp4Tensor, _type


class _MoeArgs(C.Structure):
    _fields_ = [("type", C.c_int), ("tokens", C.c_int), ("top_k", C.c_int), ("renormalize", C.c_int), ("x", C.c_void_p),
                ("ldx", C.c_longlong), ("router", C.c_void_p), ("ld_router", C.c_longlong), ("gate_up", _Fp4Tensor),
                ("down", _Fp4Tensor), ("y", C.c_void_p), ("ldy", C.c_longlong), ("chosen", C.c_void_p), ("weights", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


def moe_workspace_bytes(tokens: int, experts: int, top_k: int, d: int, f: int) -> int:
    """mcd_moe_workspace; 0 for sizes that mcd_moe_layer refuses."""
    return lib().mcd_moe_workspace(tokens, experts, top_k, d, f)


class MoeLayer:
    """mcd_moe_layer: a router and gated experts with 4-bit weights on a few tokens, kept for any number of enqueue() calls.

    gate_up: batch = experts, rows = 2f (f of the gate, then f of the up projection), cols = d; down: rows = d, cols = f."""

    def __init__(self, gate_up: Fp4Matrix, down: Fp4Matrix, x: int, dtype: str, router: int, y: int, *, tokens: int, top_k: int,
                 renormalize: bool = True, ldx: int = 0, ld_router: int = 0, ldy: int = 0, chosen: int = 0, weights: int = 0,
                 workspace: int = 0, workspace_bytes: int = 0):
        d = gate_up.cols
        self._args = _MoeArgs(_type(dtype), tokens, top_k, 1 if renormalize else 0, x or None, ldx or d, router or None, ld_router or d,
                              gate_up._c, down._c, y or None, ldy or d, chosen or None, weights or None, workspace or None,
                              workspace_bytes)
        self._ref = C.byref(self._args)
        self._call = lib().mcd_moe_layer

    def enqueue(self, stream: int = 0) -> None:
        _check(self._call(self._ref, stream))
