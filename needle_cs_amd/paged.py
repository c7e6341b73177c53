"""An int8 KV cache in pages (``nhip_paged_*``; no counterpart in the reference).

``PagedCache`` holds the arrays of one cache, or the addresses of a caller's
own, and makes the library's calls on them.  Arguments named as addresses
(``q``, ``row_seq``, ``workspace``, ...) are device pointers; every call is
asynchronous on ``stream`` (an address; None: the library's stream) and can be
captured in a graph.  include/needle_hip.h says what each call does.
"""
from __future__ import annotations

import ctypes as C

from . import DeviceBuffer, check, lib


class PagedCacheView(C.Structure):
    """nhip_paged_cache."""
    _fields_ = [("keys", C.c_void_p), ("key_scales", C.c_void_p), ("values", C.c_void_p),
                ("value_scales", C.c_void_p), ("tables", C.c_void_p), ("lengths", C.c_void_p), ("refs", C.c_void_p),
                ("layers", C.c_int32), ("pages", C.c_int32), ("page_size", C.c_int32), ("kv_heads", C.c_int32),
                ("qk_dim", C.c_int32), ("v_dim", C.c_int32), ("sequences", C.c_int32), ("width", C.c_int32)]


class PagedCache:
    """A paged cache: of its own memory, empty, or over ``buffers`` (device
    pointers by the names of the view's arrays, as they stand)."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, qk_dim: int, v_dim: int,
                 sequences: int, width: int, buffers: dict | None = None):
        self.buffers = {}
        if buffers is None:
            cells = layers * pages * kv_heads * page_size
            sizes = {"keys": cells * qk_dim, "key_scales": 4 * cells, "values": cells * v_dim,
                     "value_scales": 4 * cells, "tables": 4 * sequences * width, "lengths": 4 * sequences,
                     "refs": 4 * pages}
            if min(layers, pages, page_size, kv_heads, qk_dim, v_dim, sequences, width) <= 0:
                raise ValueError("a paged cache's sizes are positive")
            self.buffers = {name: DeviceBuffer(size) for name, size in sizes.items()}
            buffers = {name: b.ptr for name, b in self.buffers.items()}
        self.view = PagedCacheView(layers=layers, pages=pages, page_size=page_size, kv_heads=kv_heads, qk_dim=qk_dim,
                                   v_dim=v_dim, sequences=sequences, width=width, **buffers)
        self.ptr = C.addressof(self.view)
        if self.buffers:
            self.reset()
            check(lib().nhip_stream_sync(None))  # calls on any stream find it empty

    def reset(self, stream=None) -> None:
        check(lib().nhip_paged_reset_dev(self.ptr, stream))

    def append(self, layer: int, k, ldk: int, v, ldv: int, row_seq, row_pos, rows: int, stream=None) -> None:
        check(lib().nhip_paged_append_dev(self.ptr, layer, k, ldk, v, ldv, row_seq, row_pos, rows, stream))

    def rotary_append(self, layer: int, rotary, q, ldq: int, heads: int, k, ldk: int, v, ldv: int, row_seq, row_pos,
                      rows: int, codes, q_scales, stream=None) -> None:
        """`rotary`: a ``needle_cs_amd.rotary.Rotary``."""
        check(lib().nhip_paged_rotary_append_dev(self.ptr, layer, rotary.ptr, q, ldq, heads, k, ldk, v, ldv, row_seq,
                                                 row_pos, rows, codes, q_scales, stream))

    def read(self, layer: int, row_seq, row_pos, rows: int, k, ldk: int, v, ldv: int, stream=None) -> None:
        check(lib().nhip_paged_read_dev(self.ptr, layer, row_seq, row_pos, rows, k, ldk, v, ldv, stream))

    def decode_workspace(self, rows: int, heads: int, max_count: int) -> int:
        return lib().nhip_paged_decode_workspace(self.ptr, rows, heads, max_count)

    def decode(self, layer: int, q, q_scales, rows: int, heads: int, row_seq, row_first, row_count, max_count: int,
               workspace, workspace_bytes: int, out, stream=None) -> None:
        check(lib().nhip_paged_decode_dev(self.ptr, layer, q, q_scales, rows, heads, row_seq, row_first, row_count,
                                          max_count, workspace, workspace_bytes, out, stream))

    def prompt_workspace(self, rows: int, heads: int, runs: int, max_count: int) -> int:
        return lib().nhip_paged_prompt_workspace(self.ptr, rows, heads, runs, max_count)

    def prompt(self, layer: int, q, q_scales, rows: int, heads: int, runs: int, run_rows, run_seq, run_pos,
               window: int, max_count: int, workspace, workspace_bytes: int, out, stream=None) -> None:
        check(lib().nhip_paged_prompt_dev(self.ptr, layer, q, q_scales, rows, heads, runs, run_rows, run_seq, run_pos,
                                          window, max_count, workspace, workspace_bytes, out, stream))

    def decode_sinks_workspace(self, rows: int, heads: int, sinks: int, max_count: int) -> int:
        return lib().nhip_paged_decode_sinks_workspace(self.ptr, rows, heads, sinks, max_count)

    def decode_sinks(self, layer: int, q, q_scales, rows: int, heads: int, row_seq, row_first, row_count, sinks: int,
                     max_count: int, workspace, workspace_bytes: int, out, stream=None) -> None:
        check(lib().nhip_paged_decode_sinks_dev(self.ptr, layer, q, q_scales, rows, heads, row_seq, row_first,
                                                row_count, sinks, max_count, workspace, workspace_bytes, out, stream))

    def prompt_sinks_workspace(self, rows: int, heads: int, runs: int, sinks: int, max_count: int) -> int:
        return lib().nhip_paged_prompt_sinks_workspace(self.ptr, rows, heads, runs, sinks, max_count)

    def prompt_sinks(self, layer: int, q, q_scales, rows: int, heads: int, runs: int, run_rows, run_seq, run_pos,
                     window: int, sinks: int, max_count: int, workspace, workspace_bytes: int, out,
                     stream=None) -> None:
        check(lib().nhip_paged_prompt_sinks_dev(self.ptr, layer, q, q_scales, rows, heads, runs, run_rows, run_seq,
                                                run_pos, window, sinks, max_count, workspace, workspace_bytes, out,
                                                stream))

    def pages_workspace(self, count: int) -> int:
        return lib().nhip_paged_pages_workspace(self.ptr, count)

    def copy(self, count: int, src, dst, stream=None) -> None:
        check(lib().nhip_paged_copy_dev(self.ptr, count, src, dst, stream))

    def fork(self, count: int, dst, src, length, workspace, workspace_bytes: int, stream=None) -> None:
        check(lib().nhip_paged_fork_dev(self.ptr, count, dst, src, length, workspace, workspace_bytes, stream))

    def resize(self, count: int, seq, length, status, workspace, workspace_bytes: int, stream=None) -> None:
        check(lib().nhip_paged_resize_dev(self.ptr, count, seq, length, status, workspace, workspace_bytes, stream))

    def free(self, count: int, seq, workspace, workspace_bytes: int, stream=None) -> None:
        check(lib().nhip_paged_free_dev(self.ptr, count, seq, workspace, workspace_bytes, stream))

    def compact(self, status, workspace, workspace_bytes: int, stream=None) -> None:
        check(lib().nhip_paged_compact_dev(self.ptr, status, workspace, workspace_bytes, stream))

    def close(self) -> None:
        """Frees the cache's own memory; later calls are refused."""
        for name in ("keys", "key_scales", "values", "value_scales", "tables", "lengths", "refs"):
            setattr(self.view, name, None)
        for b in self.buffers.values():
            b.close()
        self.buffers = {}
