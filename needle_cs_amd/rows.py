"""Row operations between a layer's int8 products (``nhip_add_rms_quantize_dev``,
``nhip_dequantize_rows_dev``; no counterpart in the reference).  Arrays are
device pointers; calls are asynchronous on ``stream`` (an address; None: the
library's stream).  include/needle_hip.h says what each does.
"""
from __future__ import annotations

from . import check, lib


def add_rms_quantize(x, ldx: int, delta, ldd: int, gain, zero_centered: bool, eps: float, rows: int, cols: int, total,
                     ld_total: int, q, scales, stream=None) -> None:
    """`total` takes x + delta (None: it is not kept)."""
    check(lib().nhip_add_rms_quantize_dev(x, ldx, delta, ldd, gain, zero_centered, eps, rows, cols, total, ld_total, q,
                                          scales, stream))


def dequantize_rows(q, scales, rows: int, cols: int, x, ldx: int, stream=None) -> None:
    check(lib().nhip_dequantize_rows_dev(q, scales, rows, cols, x, ldx, stream))
