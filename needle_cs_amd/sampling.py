"""Token ids drawn from logits (``nhip_sample_dev``; no counterpart in the
reference, which takes the largest).  Arrays are device pointers; calls are
asynchronous on ``stream`` (an address; None: the library's stream).
include/needle_hip.h says what is kept and drawn.
"""
from __future__ import annotations

import ctypes as C

from . import check, lib


class Sampling(C.Structure):
    """nhip_sampling: a number in [0, 1) and the settings of every row (None: every row's default)."""
    _fields_ = [("random", C.c_void_p), ("temperature", C.c_void_p), ("top_k", C.c_void_p), ("top_p", C.c_void_p),
                ("min_p", C.c_void_p)]


def sample_workspace(rows: int, n: int) -> int:
    return lib().nhip_sample_workspace(rows, n)


def sample(logits, ldx: int, n: int, rows: int, sampling: Sampling, mask, mask_ld: int, words: int, workspace,
           workspace_bytes: int, ids, logprobs, stream=None) -> None:
    """`mask` None: every id; `logprobs` None: not wanted."""
    check(lib().nhip_sample_dev(logits, ldx, n, rows, C.addressof(sampling), mask, mask_ld, words, workspace,
                                workspace_bytes, ids, logprobs, stream))
