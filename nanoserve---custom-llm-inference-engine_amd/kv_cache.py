"""The paged KV cache on MI355X: new rows into their pages, and the pages themselves.

``store_kv_hip`` does in one launch what the reference's forward does between its projection and its
attention: rotate queries and keys by position (nanoserve/model/rope.py:78-91) and write keys and values
into the cache (``write_kv_to_cache``, nanoserve/model/attention.py:55-72).  It takes the batch layout that
``paged_attention_hip`` takes and finds each token's page in the block tables, so no slot list is built.

``PagePool`` keeps the pages: who holds them (the reference's ``BlockAllocator``,
nanoserve/cache/block_allocator.py:14-47, a free list on the host) is counted on the device, next to the
block tables and sequence lengths that attention reads, and rows are extended, forked, freed, released
behind a window and compacted there.  No call reads anything back, so a decode loop of ``extend``,
``store_kv_hip``, ``paged_attention_hip`` and ``release`` can be captured into a graph.

The computation runs in ``libns_kv_cache.so`` (include/ns_kv_cache.h); there is no other path: a missing
library raises.
"""
from __future__ import annotations

import contextlib
import ctypes
import os
from typing import Optional

import numpy as np
import torch

from .paged_attention import host_module

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libns_kv_cache.so")

ABI_VERSION = 1
NS_KV_DTYPE_F32 = 0
NS_KV_DTYPE_BF16 = 1
NS_KV_DTYPE_F16 = 2
MAX_ROWS = 4096           # rows of one extend or fork call (NS_KV_MAX_ROWS)
STATUS_BAD_PAGE = 1
STATUS_NO_PAGES = 2
STATUS_BAD_ROW = 4
STATUS_BAD_LENGTH = 8

EXPORTS = ("ns_kv_abi_version", "ns_kv_last_error", "ns_kv_store", "ns_kv_scratch_bytes", "ns_kv_extend", "ns_kv_fork",
           "ns_kv_free", "ns_kv_release", "ns_kv_copy", "ns_kv_compact")

_DTYPES = {torch.float32: NS_KV_DTYPE_F32, torch.bfloat16: NS_KV_DTYPE_BF16, torch.float16: NS_KV_DTYPE_F16}


class KvCacheError(RuntimeError):
    """An argument that the library or this module refused."""


class NsKvStoreArgs(ctypes.Structure):
    """ns_kv_store_args of include/ns_kv_cache.h, field for field."""

    _fields_ = ([(n, ctypes.c_void_p) for n in
                 ("query", "key", "value", "k_cache", "v_cache", "out", "inv_freq", "block_tables", "seq_lens",
                  "query_start_loc", "query_lens", "status")]
                + [(n, ctypes.c_int64) for n in
                   ("stride_q_token", "stride_q_head", "stride_key_token", "stride_key_head", "stride_value_token",
                    "stride_value_head", "stride_k_block", "stride_k_token", "stride_k_head", "stride_v_block",
                    "stride_v_token", "stride_v_head", "stride_o_token", "stride_o_head", "stride_bt_seq")]
                + [(n, ctypes.c_int32) for n in
                   ("total", "num_seqs", "num_heads_q", "num_kv_heads", "head_dim", "block_size", "num_blocks",
                    "max_blocks_per_seq", "dtype")])


class NsKvPool(ctypes.Structure):
    """ns_kv_pool of include/ns_kv_cache.h, field for field."""

    _fields_ = ([(n, ctypes.c_void_p) for n in
                 ("block_tables", "seq_lens", "page_refs", "status", "tensors", "scratch")]
                + [("scratch_bytes", ctypes.c_uint64), ("stride_bt_row", ctypes.c_int64), ("slot_bytes", ctypes.c_int64)]
                + [(n, ctypes.c_int32) for n in ("num_rows", "num_cols", "num_pages", "num_tensors", "block_size")])


_LIB: Optional[ctypes.CDLL] = None
_STORE = None    # the host module's function, and the addresses of the library's that it calls
_PAGES = None    # the same for the pool's: the function, ns_kv_last_error, and the others by name


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load the HIP library (raises when it is not built: there is no fallback)."""
    global _LIB, _STORE, _PAGES
    if _LIB is not None:
        return _LIB
    if not os.path.exists(path):
        raise KvCacheError(f"{path} is not built (run __graft_entry__.build())")
    lib = ctypes.CDLL(path)
    p, i, pool = ctypes.c_void_p, ctypes.c_int32, ctypes.POINTER(NsKvPool)
    for name, args in (("ns_kv_abi_version", []), ("ns_kv_last_error", []),
                       ("ns_kv_store", [ctypes.POINTER(NsKvStoreArgs), p]),
                       ("ns_kv_scratch_bytes", [i, ctypes.POINTER(ctypes.c_uint64)]),
                       ("ns_kv_extend", [pool, p, p, i, p]), ("ns_kv_fork", [pool, p, p, i, p]),
                       ("ns_kv_free", [pool, p, i, p]), ("ns_kv_release", [pool, p, i, i, i, p]),
                       ("ns_kv_copy", [pool, pool, p, p, i, p]), ("ns_kv_compact", [pool, pool, p, p])):
        f = getattr(lib, name)
        f.restype, f.argtypes = ctypes.c_int, args
    lib.ns_kv_last_error.restype = ctypes.c_char_p
    if lib.ns_kv_abi_version() != ABI_VERSION:
        raise KvCacheError(f"ABI {lib.ns_kv_abi_version()} in {path}, expected {ABI_VERSION}")
    host = host_module(KvCacheError)
    host.set_errors(None, KvCacheError)
    _STORE = (host.store, *(ctypes.cast(f, p).value for f in (lib.ns_kv_store, lib.ns_kv_last_error)))
    _PAGES = (host.pages, _STORE[2], {n: ctypes.cast(getattr(lib, "ns_kv_" + n), p).value
                                      for n in ("free", "extend", "fork", "release")})
    _LIB = lib
    return lib


def _check(rc: int) -> None:
    if rc != 0:
        raise KvCacheError(load().ns_kv_last_error().decode())


_NO_SWITCH = contextlib.nullcontext()


def _on(dev: int, stream):
    """(HIP stream handle, context) of a call on device ``dev``: its current stream, a torch stream or a raw handle (0:
    the default stream).  Inside the context the call's temporaries are made on that stream."""
    if stream is None:
        if dev == torch.cuda.current_device():
            return torch._C._cuda_getCurrentRawStream(dev), _NO_SWITCH
        s = torch.cuda.current_stream(dev)
    elif isinstance(stream, torch.cuda.Stream):
        if stream.device_index != dev:
            raise KvCacheError(f"the stream is one of device {stream.device_index}, the tensors are on device {dev}")
        s = stream
    elif int(stream) == 0:
        s = torch.cuda.default_stream(dev)
    else:
        s = torch.cuda.ExternalStream(int(stream), device=dev)
    return s.cuda_stream, torch.cuda.stream(s)


def _i32(t, dev, name):
    if t.dtype is torch.int32 and t.device == dev and t.is_contiguous():
        return t
    if t.is_floating_point() or t.is_complex() or t.dtype is torch.bool:
        raise KvCacheError(f"{name} must be an integer tensor")
    return t.to(device=dev, dtype=torch.int32).contiguous()


def _pieces(t):
    """(address, bytes from piece to piece, pieces, bytes of a piece) of a tensor whose entries t[i] are contiguous."""
    size, n = t.element_size(), t.shape[0]
    if n and t.is_contiguous():
        return t.data_ptr(), t.numel() * size, 1, t.numel() * size
    return t.data_ptr(), t.stride(0) * size, n, t[0].numel() * size if n else 0


def _overlap(a, b):
    """Whether two tensors, given by their ``_pieces``, have a byte in common (slices of one tensor may lie between
    each other and have none)."""
    (a0, step_a, na, la), (b0, step_b, nb, lb) = a, b
    if min(na, nb, la, lb) < 1 or a0 + (na - 1) * step_a + la <= b0 or b0 + (nb - 1) * step_b + lb <= a0:
        return False
    if na == 1 or nb == 1 or step_a != step_b:
        if na < nb:
            a0, step_a, na, la, b0, step_b, nb, lb = b0, step_b, nb, lb, a0, step_a, na, la
        # for each piece of b: the last of a that begins below its end
        b = b0 + step_b * np.arange(nb, dtype=np.int64)
        i = np.minimum((b + lb - 1 - a0) // step_a, na - 1)
        return bool(((i >= 0) & (a0 + i * step_a + la > b)).any())
    # of one step: piece i of a meets piece i + k of b for the k that bring them nearest
    near = (a0 - b0) // step_a
    return any(-na < k < nb and a0 < b0 + k * step_a + lb and b0 + k * step_a < a0 + la for k in (near, near + 1))


class _Memory:
    """What a pool's caches and tables occupy."""

    def __init__(self, caches, tables):
        self.caches, self.tables = [_pieces(t) for t in caches], [_pieces(t) for t in tables]
        self.low = np.array([at for at, _, _, _ in self.caches])
        self.high = np.array([at + step * (n - 1) + size for at, step, n, size in self.caches])
        self.lows, self.highs = np.sort(self.low), np.sort(self.high)

    def shared_cache(self, other):
        # of each cache here, how many there begin before its end and do not end before its beginning: mostly none,
        # which takes 5 us for 56 caches each, where looking at all pairs takes 3 ms
        near = np.searchsorted(other.lows, self.high) - np.searchsorted(other.highs, self.low, "right")
        return near.any() and any(_overlap(a, b) for a, n in zip(self.caches, near) if n for b in other.caches)

    def shared_table(self, other):
        return any(map(_overlap, self.tables, other.tables))


def store_kv_hip(key, value, k_cache, v_cache, block_tables, seq_lens, query_start_loc, query_lens, block_size: int, *,
                 query=None, inv_freq=None, out=None, status=None, stream=None):
    """Writes the new tokens' keys and values into their pages; with ``inv_freq``, keys and ``query`` are rotated by
    position.  Returns the rotated query (``out`` if given), or None without one.

    key, value (total, Hkv, D) of the caches' dtype (views into a fused projection are taken as they are);
    k_cache, v_cache (num_blocks, block_size, Hkv, D); block_tables, seq_lens (lengths that include the new tokens),
    query_start_loc, query_lens and block_size as ``paged_attention_hip`` takes them: a token's position, and so its
    page and slot, is the one that attention gives it.  Rows that are no sequence's token are left alone.  Two tokens
    of a call are not to share a page and slot.

    inv_freq (D / 2) float32: element j and element j + D / 2 of a head are turned by position * inv_freq[j] (the
    reference's rotate-half form), the angle formed in 64 bits.  ``query`` (total, Hq, D) needs it.  ``out``: where
    the rotated query goes, ``query`` itself for in place.  ``status``: an int32 device tensor of one element that
    STATUS_BAD_PAGE is ORed into when a token has no valid page (its row is then not stored).  ``stream``: a
    ``torch.cuda.Stream`` or a raw handle, default the current stream.
    """
    if _STORE is None:
        load()
    store, entry, why = _STORE
    dev = k_cache.get_device()
    if dev < 0:
        handle, on = -1, _NO_SWITCH      # checked, and refused
    elif stream is None and dev == torch.cuda.current_device():
        return store(entry, why, key, value, k_cache, v_cache, block_tables, seq_lens, query_start_loc, query_lens,
                     block_size, query, inv_freq, out, status, torch._C._cuda_getCurrentRawStream(dev))
    else:
        handle, on = _on(dev, stream)
    with on:
        return store(entry, why, key, value, k_cache, v_cache, block_tables, seq_lens, query_start_loc, query_lens,
                     block_size, query, inv_freq, out, status, handle)


class PagePool:
    """The pages of a paged cache and the sequences that hold them, all on the device.

    k_caches, v_caches: the layers' tensors, (pages, block_size, Hkv, D) each, any dtype, a page contiguous.
    block_tables (rows, columns) int32, seq_lens (rows) int32: row r holds ``seq_lens[r]`` tokens in the pages
    ``block_tables[r, : ceil(seq_lens[r] / block_size)]``, -1 for one released behind a window.  page_refs (pages)
    int32: how many table entries name each page, plus one for a page that is never handed out; 0: free.  The pool
    works on the tensors given, which ``paged_attention_hip`` and ``store_kv_hip`` take as they are;
    ``PagePool.empty`` makes them.

    The rows that a method takes are int32 tensors on the pool's device (or sequences of ints, which are copied
    there).  What a call cannot do is left undone and marked in ``status``, an int32 device tensor of STATUS_* bits
    that the caller reads (and clears) when it wants: NO_PAGES, BAD_ROW (no such row, listed twice, or not empty),
    BAD_LENGTH, BAD_PAGE.  Results do not depend on timing: pages are handed out lowest first, in the order of
    the list.  One pool's calls run one after another; ``stream`` as in ``store_kv_hip``.  A pool may be dropped while
    calls on torch's streams run: its tensors stay allocated until these have ended.  It is kept until calls on a
    stream given as a raw handle have ended, and as long as graphs that hold its calls are replayed.
    """

    def __init__(self, k_caches, v_caches, block_tables, seq_lens, page_refs):
        caches = list(k_caches) + list(v_caches)
        if len(k_caches) != len(v_caches) or not caches:
            raise KvCacheError("a pool needs as many k_caches as v_caches, at least one")
        first = caches[0]
        if first.dim() != 4:
            raise KvCacheError("caches must be (pages, block_size, heads, head_dim)")
        for c in caches:
            if c.shape != first.shape or c.dtype is not first.dtype or c.device != first.device:
                raise KvCacheError("all caches of a pool must share shape, dtype and device")
            if not c[:1].is_contiguous():
                raise KvCacheError("a cache's pages must be contiguous")
            if c.shape[0] > 1 and c.stride(0) < c[0].numel():
                raise KvCacheError("a cache's pages overlap")
        pages, bs, heads, d = first.shape
        if block_tables.dim() != 2:
            raise KvCacheError("block_tables must be (rows, columns) with contiguous rows")
        dev, slot = first.device, heads * d * first.element_size()
        if min(pages, bs) < 1 or slot < 16 or slot % 16 != 0:
            raise KvCacheError(f"a page's slot must be a positive multiple of 16 bytes (got {slot})")
        for name, t, shape in (("block_tables", block_tables, None), ("seq_lens", seq_lens, (block_tables.shape[0],)),
                               ("page_refs", page_refs, (pages,))):
            if t.dtype is not torch.int32 or t.device != dev or (shape is not None and t.shape != shape):
                raise KvCacheError(f"{name} must be an int32 tensor on the caches' device"
                                   + (f" of shape {shape}" if shape is not None else ""))
        if block_tables.numel() == 0 or block_tables.stride(1) != 1 \
                or block_tables.stride(0) < block_tables.shape[1]:
            raise KvCacheError("block_tables must be (rows, columns) with contiguous rows")
        if not seq_lens.is_contiguous() or not page_refs.is_contiguous():
            raise KvCacheError("seq_lens and page_refs must be contiguous")
        if any(c.data_ptr() % 16 or c.stride(0) * c.element_size() % 16 for c in caches):
            raise KvCacheError("pages must be 16-byte aligned")
        if dev.type != "cuda":
            raise KvCacheError("PagePool needs device tensors")
        self._lib = load()
        need = ctypes.c_uint64(0)
        _check(self._lib.ns_kv_scratch_bytes(pages, ctypes.byref(need)))
        self.k_caches, self.v_caches = list(k_caches), list(v_caches)
        self.block_tables, self.seq_lens, self.page_refs = block_tables, seq_lens, page_refs
        self.device, self.block_size, self.num_pages = dev, bs, pages
        self._dev = first.get_device()
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._scratch = torch.empty(int(need.value), dtype=torch.uint8, device=dev)
        # (a copy from pageable memory: once it returns, the tensors made before it can be used on any stream)
        self._tensors = torch.tensor([[c.data_ptr(), c.stride(0) * c.element_size()] for c in caches],
                                     dtype=torch.int64, device=dev)
        self._pool = NsKvPool(block_tables.data_ptr(), seq_lens.data_ptr(), page_refs.data_ptr(), self.status.data_ptr(),
                              self._tensors.data_ptr(), self._scratch.data_ptr(), int(need.value),
                              block_tables.stride(0), slot, block_tables.shape[0], block_tables.shape[1], pages,
                              len(caches), bs)
        self._ref, self._at = ctypes.byref(self._pool), ctypes.addressof(self._pool)
        self._memory = _Memory(caches, (block_tables, seq_lens, page_refs))
        self._streams = set()    # handles of the torch streams that the tensors are recorded on

    @classmethod
    def empty(cls, k_caches, v_caches, max_seqs: int, max_pages_per_seq: int, reserved: int = 1):
        """A pool of no sequences over the caches.  The first ``reserved`` pages are never handed out (the reference
        keeps page 0 for padding)."""
        dev, pages = k_caches[0].device, k_caches[0].shape[0]
        refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        refs[:reserved] = 1
        return cls(k_caches, v_caches, torch.full((max_seqs, max_pages_per_seq), -1, dtype=torch.int32, device=dev),
                   torch.zeros(max_seqs, dtype=torch.int32, device=dev), refs)

    def _on(self, stream):
        """``_on`` of a call of this pool, whose tensors are recorded on the call's stream."""
        handle, on = _on(self._dev, stream)
        if handle not in self._streams and (stream is None or isinstance(stream, torch.cuda.Stream)):
            self._record(handle, torch.cuda.current_stream(self.device) if stream is None else stream)
        return handle, on

    def _record(self, handle, stream):
        for t in (*self.k_caches, *self.v_caches, self.block_tables, self.seq_lens, self.page_refs, self.status,
                  self._scratch, self._tensors):
            t.record_stream(stream)
        self._streams.add(handle)

    def _list(self, x, name):
        if isinstance(x, torch.Tensor) and x.dtype is torch.int32 and x.dim() == 1 and x.get_device() == self._dev \
                and x.is_contiguous():
            return x
        if not isinstance(x, torch.Tensor):
            x = torch.tensor(list(x), dtype=torch.int32)
        if x.dim() != 1:
            raise KvCacheError(f"{name} must have one dimension")
        return _i32(x, self.device, name)

    def _two(self, a, b, names):
        a, b = self._list(a, names[0]), self._list(b, names[1])
        if a.numel() != b.numel():
            raise KvCacheError(f"{names[0]} and {names[1]} must be as many (got {a.numel()} and {b.numel()})")
        return a, b

    def _change(self, kind, name, a, b, names, window, sinks, stream):
        """One of the calls that change the tables."""
        pages, why, entries = _PAGES
        dev = self._dev
        if stream is None and dev == torch.cuda.current_device():
            handle = torch._C._cuda_getCurrentRawStream(dev)
            if handle in self._streams and pages(kind, entries[name], why, self._at, dev, a, b, window, sinks,
                                                 handle) is None:
                return
        handle, on = self._on(stream)
        with on:   # the lists are made on the call's stream
            if b is None:
                a = self._list(a, names[0])
            else:
                a, b = self._two(a, b, names)
            if pages(kind, entries[name], why, self._at, dev, a, b, window, sinks, handle) is not None:
                raise KvCacheError(f"{' and '.join(names)} must be lists of rows")

    def extend(self, rows, lens, stream=None) -> None:
        """Row ``rows[i]`` grows to ``lens[i]`` tokens (its length grows with it) and gets the pages for them, the
        lowest free ones first.  A row is served if the pages that it and the rows listed before it ask for are all
        there, or if it asks for none; else it is left as it was (NO_PAGES).  At most MAX_ROWS rows a call."""
        self._change(1, "extend", rows, lens, ("rows", "lens"), 0, 0, stream)

    def fork(self, parents, children, stream=None) -> None:
        """Row ``children[i]``, an empty one, becomes a copy of row ``parents[i]``: full pages are shared, the tokens
        of a last page that is not full are copied, in every layer, to a page of the child's own.  A child for which
        no page is left stays empty (NO_PAGES).  At most MAX_ROWS pairs a call."""
        self._change(1, "fork", parents, children, ("parents", "children"), 0, 0, stream)

    def free(self, rows, stream=None) -> None:
        """The rows give up their pages and become empty; a page that no row names any more is free."""
        self._change(0, "free", rows, None, ("rows",), 0, 0, stream)

    def release(self, rows, window: int, sinks: int = 0, stream=None) -> None:
        """The rows give up the pages that no later token sees through ``window`` and ``sinks`` (those of
        ``paged_attention_hip``); their entries become -1."""
        if not 1 <= window < 2 ** 31:
            raise KvCacheError(f"window must be at least 1 and below 2^31 (got {window})")
        if not 0 <= sinks < 2 ** 31:
            raise KvCacheError(f"sinks must lie in [0, 2^31) (got {sinks})")
        self._change(2, "release", rows, None, ("rows",), window, sinks, stream)

    def copy(self, src, dst, into: Optional["PagePool"] = None, stream=None) -> None:
        """Pages ``src[i]`` to pages ``dst[i]``, in every layer, of this pool or of ``into``, a pool of pages alike.
        No page is to be in ``dst`` twice or, within one pool, in both lists (checked for lists, not for tensors).
        Tables and counts stay as they are."""
        to = self if into is None else into
        self._alike(to)
        if not isinstance(dst, torch.Tensor):
            dst = list(dst)
            other = []
            if to is self and not isinstance(src, torch.Tensor):
                other = src = list(src)
            if len(set(dst)) != len(dst) or set(other) & set(dst):
                raise KvCacheError("a page is named twice by dst, or by src and dst")
        handle, on = self._on(stream)
        if to is not self:
            to._on(stream)
        with on:
            src, dst = self._two(src, dst, ("src", "dst"))
            _check(self._lib.ns_kv_copy(self._ref, to._ref, src.data_ptr(), dst.data_ptr(), src.numel(), handle))

    def compact(self, stream=None):
        """Moves the pages in use to the lowest numbers: with m in use, those numbered m or higher go, in ascending
        order, to the free ones below m; tables and counts follow.  Returns page_map (pages) int32, each page's new
        number, -1 for a free one."""
        return self._compact(None, stream)

    def compact_into(self, to: "PagePool", stream=None):
        """As ``compact``, but the pages in use go to the numbers below m of ``to``, another pool (a smaller one, say)
        of as many rows, columns and layers, whose tables, lengths and counts are overwritten; this pool stays as it
        is.  A ``to`` of fewer than m pages is left alone (NO_PAGES, and a page_map of -1)."""
        if to is self:
            raise KvCacheError("compact_into takes another pool")
        self._alike(to)
        if to.block_tables.shape != self.block_tables.shape:
            raise KvCacheError("the pools' block tables differ in shape")
        if self._memory.shared_cache(to._memory):
            raise KvCacheError("the pools share a cache")
        if self._memory.shared_table(to._memory):
            raise KvCacheError("the pools share a table")
        return self._compact(to, stream)

    def _alike(self, to):
        if to is self:
            return
        a, b = self.k_caches[0], to.k_caches[0]
        if len(self.k_caches) != len(to.k_caches) or a.shape[1:] != b.shape[1:] or a.dtype is not b.dtype \
                or self.device != to.device:
            raise KvCacheError("the pools' caches differ in layers, page shape, dtype or device")

    def _compact(self, to, stream):
        handle, on = self._on(stream)
        if to is not None:
            to._on(stream)
        with on:
            page_map = torch.empty(self.num_pages, dtype=torch.int32, device=self.device)
            _check(self._lib.ns_kv_compact(self._ref, to._ref if to is not None else None, page_map.data_ptr(), handle))
        return page_map
