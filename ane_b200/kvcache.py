"""Paged key/value cache of a decode loop, all of it in device memory.

`KVCache` holds two pools of pages (K and V, [layers, pages, page_tokens,
kv_heads, dim], float16 or bfloat16), a count of readers per page (`refs`, 0 =
free), and per slot a row of page numbers (`tables`) and a token count (`lens`).
Sequences grow (`reserve`, then `write` on each layer), are forked for several
continuations of one prompt (`fork`: whole pages are shared, the part page is
copied), are freed, and the pool is compacted to give its tail back.  No call
waits for the host, so a loop of them can be captured in a CUDA graph; a request
that finds no free pages is reported in `granted` and changes nothing.

The reference has no cache of its own (its ggml backend leaves attention to
ggml): the operations are declared in include/ane_b200.h.
"""
from __future__ import annotations

import ctypes

import torch

import ane_b200 as ane


class _Desc(ctypes.Structure):
    """ane_kv_cache (include/ane_b200.h)."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("dtype", ctypes.c_uint32), ("layers", ctypes.c_uint32),
                ("pages", ctypes.c_uint32), ("page_tokens", ctypes.c_uint32), ("heads", ctypes.c_uint32),
                ("dim", ctypes.c_uint32), ("refs", ctypes.c_void_p), ("tables", ctypes.c_void_p),
                ("lens", ctypes.c_void_p), ("slots", ctypes.c_uint32), ("max_pages", ctypes.c_uint32),
                ("ctl", ctypes.c_void_p)]


class KVCache:
    def __init__(self, k, v, refs, tables, lens):
        """Takes the cache's tensors: pools k and v, refs int32 [pages], tables
        int32 [slots, max_pages], lens int32 [slots] (zeros for a new cache)."""
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype or not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("k and v must be contiguous [layers, pages, page_tokens, kv_heads, dim] of one type")
        if k.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError("a cache holds float16 or bfloat16, got %s" % k.dtype)
        layers, pages, page_tokens, heads, dim = k.shape
        if refs.shape != (pages,) or tables.dim() != 2 or lens.shape != (tables.shape[0],):
            raise ValueError("refs must be [pages], tables [slots, max_pages], lens [slots]")
        for name, t in (("refs", refs), ("tables", tables), ("lens", lens)):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != k.device:
                raise ValueError("%s must be a contiguous int32 tensor on the pools' device" % name)
        if v.device != k.device:
            raise ValueError("k and v must be on one device")
        self.k, self.v, self.refs, self.tables, self.lens = k, v, refs, tables, lens
        self.layers, self.pages, self.page_tokens, self.kv_heads, self.dim = layers, pages, page_tokens, heads, dim
        self.slots, self.max_pages = tables.shape
        self._ctl = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._desc = _Desc(k.data_ptr(), v.data_ptr(), ane._dtype(k), layers, pages, page_tokens, heads, dim,
                           refs.data_ptr(), tables.data_ptr(), lens.data_ptr(), self.slots, self.max_pages,
                           self._ctl.data_ptr())
        self._ref = ctypes.byref(self._desc)
        self._device = ane._device(k)

    @classmethod
    def empty(cls, layers: int, pages: int, page_tokens: int, kv_heads: int, dim: int, slots: int, max_pages: int,
              dtype=torch.float16, device="cuda") -> "KVCache":
        """A new cache without sequences."""
        shape = (layers, pages, page_tokens, kv_heads, dim)
        ints = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)  # noqa: E731
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                   ints(pages), ints(slots, max_pages), ints(slots))

    def _granted(self, granted, n, stream):
        if granted is None:
            granted = self._new(n, stream)
        return granted

    def _new(self, n, stream):
        return ane._made_for(stream, lambda: torch.empty(n, dtype=torch.int32, device=self.k.device))

    def reserve(self, slots, counts, granted=None, stream=None):
        """Grows slots[i] by counts[i] tokens; returns granted (int32, 1 or 0)."""
        n, dev = slots.numel(), self._device
        granted = self._granted(granted, n, stream)
        ane.check(ane.lib.ane_kv_reserve_dev(self._ref, n, ane._i32_vector("slots", slots, dev),
                                             ane._i32_vector("counts", counts, dev, n),
                                             ane._i32_vector("granted", granted, dev, n), ane._stream_of(stream, dev)))
        return granted

    def write(self, layer: int, slots, k, v, cu=None, granted=None, stream=None) -> None:
        """Rows cu[i]:cu[i+1] of k and v [tokens, kv_heads, dim] (float32 or the
        cache's type; cu None: one row per slot) become the last tokens of
        slots[i] on `layer`; rows of requests that were not granted are dropped."""
        n = slots.numel()
        dev = self._device
        rk, rv = ane._rows("k", k, dev, self.kv_heads, self.dim), ane._rows("v", v, dev, self.kv_heads, self.dim)
        if k.shape[0] != v.shape[0] or k.dtype != v.dtype:
            raise ValueError("k and v must have one shape and dtype")
        ane.check(ane.lib.ane_kv_write_dev(self._ref, layer, n, ane._i32_vector("slots", slots, dev),
                                           None if cu is None else ane._i32_vector("cu", cu, dev, n + 1),
                                           None if granted is None else ane._i32_vector("granted", granted, dev, n),
                                           k.shape[0], ane._dtype(k), rk, rv,
                                           ane._stream_of(stream, dev)))

    def fork(self, parents, children, granted=None, stream=None):
        """children[i] (empty slots) become copies of parents[i]; returns granted."""
        n, dev = children.numel(), self._device
        granted = self._granted(granted, n, stream)
        ane.check(ane.lib.ane_kv_fork_dev(self._ref, n, ane._i32_vector("parents", parents, dev, n),
                                          ane._i32_vector("children", children, dev),
                                          ane._i32_vector("granted", granted, dev, n), ane._stream_of(stream, dev)))
        return granted

    def free(self, slots, stream=None) -> None:
        """The slots give up their pages and are empty."""
        ane.check(ane.lib.ane_kv_free_dev(self._ref, slots.numel(), ane._i32_vector("slots", slots, self._device),
                                          ane._stream_of(stream, self._device)))

    def copy_pages(self, src, dst, into: "KVCache | None" = None, stream=None) -> None:
        """Pages src[i] to pages dst[i] on all layers (of `into`, or of this
        cache); refs and tables are the caller's."""
        to = self if into is None else into
        n, dev = src.numel(), self._device
        if to._device != dev:
            raise ValueError("the caches are on two devices")
        ane.check(ane.lib.ane_kv_copy_pages_dev(self._ref, to._ref, n, ane._i32_vector("src", src, dev),
                                                ane._i32_vector("dst", dst, dev, n), ane._stream_of(stream, dev)))

    def compact(self, refs_out=None, tables_out=None, remap=None, live=None, stream=None):
        """Moves the pages in use to the lowest numbers.  Returns (live, remap):
        the number of pages in use (int32 [1]) and each page's new number (-1:
        free).  refs_out and tables_out default to the cache's own arrays; given
        others, the cache keeps its old state, whose pages stay intact."""
        remap = self._new(self.pages, stream) if remap is None else remap
        live = self._new(1, stream) if live is None else live
        refs_out = self.refs if refs_out is None else refs_out
        tables_out = self.tables if tables_out is None else tables_out
        dev = self._device
        if (tables_out.shape != self.tables.shape or not tables_out.is_contiguous() or
                tables_out.dtype != torch.int32 or tables_out.get_device() != dev):
            raise ValueError("tables_out must be a contiguous int32 CUDA tensor of the tables' shape on their device")
        ane.check(ane.lib.ane_kv_compact_dev(self._ref, ane._i32_vector("refs_out", refs_out, dev, self.pages),
                                             tables_out.data_ptr(), ane._i32_vector("remap", remap, dev, self.pages),
                                             ane._i32_vector("live", live, dev, 1), ane._stream_of(stream, dev)))
        return live, remap

    def attend(self, layer: int, q, slots=None, shared: int = 0, **kw):
        """ane_b200.attn_decode over one layer of this cache."""
        return ane.attn_decode(q, self.k[layer], self.v[layer], self.tables, self.lens, slots=slots, shared=shared, **kw)
