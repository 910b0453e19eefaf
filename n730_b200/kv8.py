"""The 8-bit paged key/value cache: Python calls of the ``n730_kv8_*`` functions.

``KV8Cache`` describes one layer's cache by device addresses (``include/n730_cuda.h`` has the
layout and each call's meaning); buffers belong to the caller, so torch is not required here.
A serving step with it::

    cache.append(k, v, "f16", batch, 1, lens)               # behind the cached positions
    cache.attention(q, out, "f16", batch, 1, heads, lens,   # ... and over them
                    w_in=w, w_out=w, ld_w=positions, ws=ws, ws_bytes=ws_bytes)
    # lens += 1; when a sequence outgrows its budget:
    cache.evict(batch, budget, lens, lens, w, w, pos, pos, positions, seen=seen, ws=ws2, ws_bytes=n)

Addresses are ints (0: none).  Methods raise ``N730Error`` on a negative code.
"""
from __future__ import annotations

import ctypes as C

from . import _lib

DTYPES = {"f32": 0, "f16": 1, "bf16": 2}
CODES = {"int8": 0, "e4m3": 1}


class N730KV8Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k_codes", "v_codes", "k_scales", "v_scales", "block_table")] + \
               [(n, C.c_int32) for n in ("n_pages", "max_pages", "n_kv", "head_dim", "page_size", "block", "code")]


class KV8Cache:
    """One layer's cache: code pools, scales and block table on the device."""

    def __init__(self, k_codes: int, v_codes: int, k_scales: int, v_scales: int, block_table: int, *, n_pages: int,
                 max_pages: int, n_kv: int, head_dim: int, page_size: int = 64, block: int = 16, code: str = "int8"):
        self.lib = _lib.cuda()
        self.c = N730KV8Cache(k_codes, v_codes, k_scales, v_scales, block_table, n_pages, max_pages, n_kv, head_dim,
                              page_size, block, CODES[code])
        self._ref = C.addressof(self.c)
        self.row = n_kv * head_dim

    def append(self, k: int, v: int, dtype: str, batch: int, tokens: int, lens: int, *, new: int = 0, ld: int = 0,
               stream: int = 0):
        """Rows k and v behind lens[b] cached positions; ld: elements between rows (0: packed)."""
        _lib.check(self.lib.n730_kv8_append(self._ref, k, v, DTYPES[dtype], ld or self.row, batch, tokens, lens, new,
                                            stream), "kv8_append")

    def read(self, k: int, v: int, dtype: str, batch: int, tokens: int, lens: int, *, first: int = 0, ld: int = 0,
             stream: int = 0):
        """Values of positions [first[b], first[b] + tokens) into rows k and v."""
        _lib.check(self.lib.n730_kv8_read(self._ref, k, v, DTYPES[dtype], ld or self.row, batch, tokens, first, lens,
                                          stream), "kv8_read")

    def attention_workspace(self, batch: int, tokens: int, heads: int, weights: bool = False,
                            dtype: str | None = None) -> int:
        """Bytes of the workspace that ``attention`` of this size wants (not always more for more tokens), for rows of
        any type or of ``dtype``, zeroed once by the caller; its first int32 is 1 after a device wait ran out."""
        if dtype is not None:
            return _lib.check(self.lib.n730_kv8_attention_ws_of(self._ref, DTYPES[dtype], batch, tokens, heads,
                                                                int(weights)), "kv8_attention_ws")
        return _lib.check(self.lib.n730_kv8_attention_ws(self._ref, batch, tokens, heads, int(weights)),
                          "kv8_attention_ws")

    def attention(self, q: int, out: int, dtype: str, batch: int, tokens: int, heads: int, lens: int, *, new: int = 0,
                  scale: float | None = None, ldq: int = 0, ldo: int = 0, w_in: int = 0, w_out: int = 0,
                  ld_w: int = 0, ws: int = 0, ws_bytes: int = 0, stream: int = 0):
        """Queries of the newest rows over the cached positions; scale defaults to head_dim ** -0.5."""
        dim = self.c.head_dim
        _lib.check(self.lib.n730_kv8_attention(self._ref, q, DTYPES[dtype], ldq or heads * dim, batch, tokens, heads,
                                               dim ** -0.5 if scale is None else scale, lens, new, out,
                                               ldo or heads * dim, w_in, w_out, ld_w, ws, ws_bytes, stream),
                   "kv8_attention")

    def evict_workspace(self, batch: int, keep: int) -> int:
        return _lib.check(self.lib.n730_kv8_evict_ws(self._ref, batch, keep), "kv8_evict_ws")

    def evict(self, batch: int, keep: int, lens: int, lens_out: int, w: int, w_out: int, pos: int, pos_out: int,
              ld_w: int, *, seen: int, first: int = 0, recent: int = 0, ws: int = 0, ws_bytes: int = 0,
              stream: int = 0):
        """Cut every longer sequence to `keep` slots per KV head by accumulated weight."""
        _lib.check(self.lib.n730_kv8_evict(self._ref, batch, keep, first, recent, seen, lens, lens_out, w, w_out, pos,
                                           pos_out, ld_w, ws, ws_bytes, stream), "kv8_evict")
