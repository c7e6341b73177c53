"""Rotary positions (``nhip_rotary_*``): tables of cos and sin, scaled for
long contexts, and heads rotated by them.  Arrays are device pointers; calls
are asynchronous on ``stream`` (an address; None: the library's stream).
include/needle_hip.h says what each does.
"""
from __future__ import annotations

import ctypes as C

from . import DeviceBuffer, check, lib

PLAIN, LINEAR, BASE, PARTS, BANDS = range(5)


class RotaryView(C.Structure):
    """nhip_rotary."""
    _fields_ = [("cos", C.c_void_p), ("sin", C.c_void_p), ("positions", C.c_int32), ("dim", C.c_int32),
                ("interleaved", C.c_int32)]


class RotaryScaling(C.Structure):
    """nhip_rotary_scaling."""
    _fields_ = [("theta", C.c_double), ("factor", C.c_double), ("low", C.c_double), ("high", C.c_double),
                ("original", C.c_double), ("magnitude", C.c_double), ("kind", C.c_int32)]


def rotary_table(cos, sin, first: int, count: int, dim: int, theta: float = 10000.0, kind: int = PLAIN,
                 factor: float = 1.0, low: float = 1.0, high: float = 32.0, original: float = 0.0,
                 magnitude: float = 1.0, stream=None) -> None:
    """Rows first .. first + count - 1 of a table into cos and sin [count][dim / 2]."""
    scaling = RotaryScaling(theta, factor, low, high, original, magnitude, kind)
    check(lib().nhip_rotary_table_dev(cos, sin, first, count, dim, C.addressof(scaling), stream))


class Rotary:
    """A table on the device and the pairs that it rotates."""

    def __init__(self, cos, sin, positions: int, dim: int, interleaved: bool = False):
        self.buffers = ()
        self.view = RotaryView(cos, sin, positions, dim, interleaved)
        self.ptr = C.addressof(self.view)

    @classmethod
    def make(cls, positions: int, dim: int, interleaved: bool = False, stream=None, **scaling) -> "Rotary":
        """With a table of its own for `positions` positions (``rotary_table``'s `scaling`), filled on `stream`."""
        if positions <= 0 or dim <= 0:
            raise ValueError("a rotary table's sizes are positive")
        buffers = DeviceBuffer(2 * positions * dim), DeviceBuffer(2 * positions * dim)
        made = cls(buffers[0].ptr, buffers[1].ptr, positions, dim, interleaved)
        made.buffers = buffers
        rotary_table(buffers[0].ptr, buffers[1].ptr, 0, positions, dim, stream=stream, **scaling)
        check(lib().nhip_stream_sync(stream))  # calls on any stream find it made
        return made

    def rotate(self, x, ldx: int, heads: int, head_dim: int, row_pos, rows: int, y, ldy: int, stream=None) -> None:
        check(lib().nhip_rotary_dev(self.ptr, x, ldx, heads, head_dim, row_pos, rows, y, ldy, stream))

    def close(self) -> None:
        """Frees a table of its own; later calls are refused."""
        self.view.cos = self.view.sin = None
        for b in self.buffers:
            b.close()
        self.buffers = ()
