"""Decoding many continuations of one prompt: Python calls of ``n730_rotary*`` and ``n730_kv16_*``.

``KV16Cache`` describes one layer's 16-bit paged cache behind a prefix that the batch shares, by device
addresses (``include/n730_cuda.h`` has the layout and each call's meaning); buffers belong to the caller,
so torch is not required here.  A decode step of a batch with it::

    turn = Rotary(freq, 128)                       # freq: frequencies(128, 1e6)[0], on the device
    cache.append(k, v, "bf16", batch, 1, lens, rotary=turn, q=q, q_out=q, heads=heads)
    cache.attention(q, out, batch, 1, heads, lens, ws=ws, ws_bytes=ws_bytes)
    # lens += 1

Addresses are ints (0: none).  Methods raise ``N730Error`` on a negative code.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from .kv8 import DTYPES

LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = {"none": 0, "linear": 1, "base": 2, "ramp": 3, "bands": 4}


class N730Rotary(C.Structure):
    _fields_ = [("d_freq", C.c_void_p), ("rotary_dim", C.c_int32), ("layout", C.c_int32), ("factor", C.c_float)]


class N730KV16Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "block_table", "prefix_table", "prefix_len")] + \
               [(n, C.c_int32) for n in ("n_pages", "max_pages", "prefix_pages", "n_kv", "head_dim", "page_size", "dtype")]


def frequencies(rotary_dim: int, theta: float = 1e4, scaling: str = "none", *, factor: float = 1.0, trained: int = 0,
                low: float = 1.0, high: float = 32.0):
    """(radians per position of each pair as float64, factor of rotated channels) for a ``Rotary``; ``low`` and
    ``high`` are turns over the ``trained`` positions (scalings "ramp" and "bands")."""
    f = np.empty(max(rotary_dim // 2, 1), np.float64)
    m = C.c_float()
    _lib.check(_lib.cuda().n730_rotary_frequencies(rotary_dim, theta, SCALINGS[scaling], factor, low, high, trained,
                                                   f.ctypes.data_as(C.c_void_p), C.byref(m)), "rotary_frequencies")
    return f, m.value


class Rotary:
    """Rotary positions: frequencies on the device, which channels pair up, the factor of rotated channels."""

    def __init__(self, freq: int, rotary_dim: int, *, layout: str = "half", factor: float = 1.0):
        self.lib = _lib.cuda()
        self.c = N730Rotary(freq, rotary_dim, LAYOUTS[layout], factor)
        self._ref = C.addressof(self.c)

    def apply(self, x: int, y: int, dtype: str, rows: int, heads: int, head_dim: int, pos: int, *, ldx: int = 0,
              ldy: int = 0, stream: int = 0):
        """Rows x of heads, rotated at positions pos[row], into rows y (y = x: in place)."""
        row = heads * head_dim
        _lib.check(self.lib.n730_rotary(self._ref, x, ldx or row, y, ldy or row, DTYPES[dtype], rows, heads, head_dim, pos,
                                        stream), "rotary")


class KV16Cache:
    """One layer's cache: pools, block table and the shared prefix's table and length, on the device."""

    def __init__(self, k: int, v: int, block_table: int, *, n_pages: int, max_pages: int, n_kv: int, head_dim: int,
                 page_size: int = 64, dtype: str = "f16", prefix_table: int = 0, prefix_pages: int = 0, prefix_len: int = 0):
        self.lib = _lib.cuda()
        self.c = N730KV16Cache(k, v, block_table, prefix_table, prefix_len, n_pages, max_pages, prefix_pages, n_kv, head_dim,
                               page_size, DTYPES[dtype])
        self._ref = C.addressof(self.c)
        self.row = n_kv * head_dim

    def append(self, k: int, v: int, dtype: str, batch: int, tokens: int, lens: int, *, new: int = 0, ld: int = 0,
               rotary: Rotary | None = None, pos: int = 0, q: int = 0, q_out: int = 0, heads: int = 0, ldq: int = 0,
               ldqo: int = 0, stream: int = 0):
        """Rows k (rotated) and v behind lens[b] cached positions; with q, its rows rotated into q_out.  All rows are of
        ``dtype``, q_out too; ``attention`` reads queries of the cache's own."""
        row = heads * self.c.head_dim
        _lib.check(self.lib.n730_kv16_append(self._ref, rotary._ref if rotary else 0, q, ldq or row, q_out, ldqo or row, heads,
                                             k, v, ld or self.row, DTYPES[dtype], batch, tokens, lens, new, pos, stream),
                   "kv16_append")

    def attention_workspace(self, batch: int, tokens: int, heads: int) -> int:
        """Bytes of the workspace that ``attention`` of this size wants, zeroed once by the caller; its first int32 is 1
        after a device wait ran out."""
        return _lib.check(self.lib.n730_kv16_attention_ws(self._ref, batch, tokens, heads), "kv16_attention_ws")

    def attention(self, q: int, out: int, batch: int, tokens: int, heads: int, lens: int, *, new: int = 0,
                  scale: float | None = None, ldq: int = 0, ldo: int = 0, ws: int = 0, ws_bytes: int = 0, stream: int = 0):
        """Queries of the newest rows, of the cache's type as out is, over the prefix and the own positions; scale defaults
        to head_dim ** -0.5."""
        dim = self.c.head_dim
        _lib.check(self.lib.n730_kv16_attention(self._ref, q, ldq or heads * dim, batch, tokens, heads,
                                                dim ** -0.5 if scale is None else scale, lens, new, out, ldo or heads * dim,
                                                ws, ws_bytes, stream), "kv16_attention")
