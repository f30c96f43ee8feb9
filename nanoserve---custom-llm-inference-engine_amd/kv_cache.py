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

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libns_kv_cache.so")

ABI_VERSION = 1
NS_KV_DTYPE_F32 = 0
NS_KV_DTYPE_BF16 = 1
NS_KV_DTYPE_F16 = 2
MAX_ROWS = 8192           # rows of one extend or fork call (NS_KV_MAX_ROWS)
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


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load the HIP library (raises when it is not built: there is no fallback)."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not os.path.exists(path):
        raise KvCacheError(f"{path} is not built (run __graft_entry__.build())")
    lib = ctypes.CDLL(path)
    p, i, pool = ctypes.c_void_p, ctypes.c_int32, ctypes.POINTER(NsKvPool)
    for name, args in (("ns_kv_abi_version", []), ("ns_kv_last_error", []),
                       ("ns_kv_store", [ctypes.POINTER(NsKvStoreArgs), p]),
                       ("ns_kv_scratch_bytes", [i, i, ctypes.POINTER(ctypes.c_uint64)]),
                       ("ns_kv_extend", [pool, p, p, i, p]), ("ns_kv_fork", [pool, p, p, i, p]),
                       ("ns_kv_free", [pool, p, i, p]), ("ns_kv_release", [pool, p, i, i, i, p]),
                       ("ns_kv_copy", [pool, pool, p, p, i, p]), ("ns_kv_compact", [pool, pool, p, p])):
        f = getattr(lib, name)
        f.restype, f.argtypes = ctypes.c_int, args
    lib.ns_kv_last_error.restype = ctypes.c_char_p
    if lib.ns_kv_abi_version() != ABI_VERSION:
        raise KvCacheError(f"ABI {lib.ns_kv_abi_version()} in {path}, expected {ABI_VERSION}")
    _LIB = lib
    return lib


def _check(rc: int) -> None:
    if rc != 0:
        raise KvCacheError(load().ns_kv_last_error().decode())


def _on(dev, stream):
    """(HIP stream handle, context) of a call: the current stream of ``dev``, a torch stream or a raw handle (0: the
    default stream).  Inside the context the call's temporaries are made on that stream."""
    if stream is None:
        s = torch.cuda.current_stream(dev)
        if dev.index == torch.cuda.current_device():
            return s.cuda_stream, contextlib.nullcontext()
    elif isinstance(stream, torch.cuda.Stream):
        s = stream
    elif int(stream) == 0:
        s = torch.cuda.default_stream(dev)
    else:
        s = torch.cuda.ExternalStream(int(stream), device=dev)
    return s.cuda_stream, torch.cuda.stream(s)


def _i32(t, dev, name):
    if t.dtype is torch.int32 and t.device == dev and t.is_contiguous():
        return t
    if t.is_floating_point() or t.is_complex():
        raise KvCacheError(f"{name} must be an integer tensor")
    return t.to(device=dev, dtype=torch.int32).contiguous()


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
    lib = load()
    dev = k_cache.device
    if key.dim() != 3 or key.shape != value.shape or k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise KvCacheError(f"key {tuple(key.shape)} and value {tuple(value.shape)} must match, and k_cache "
                           f"{tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)}")
    total, hkv, d = key.shape
    nb, bs, h, dc = k_cache.shape
    if (h, dc) != (hkv, d):
        raise KvCacheError(f"the caches' rows ({h}, {dc}) are not the keys' ({hkv}, {d})")
    if bs != block_size:
        raise KvCacheError(f"block_size {block_size} != the cache's {bs}")
    dtype = k_cache.dtype
    if dtype not in _DTYPES:
        raise KvCacheError(f"unsupported dtype {dtype} (float32, bfloat16, float16)")
    if query is None:
        if out is not None:
            raise KvCacheError("out is where the rotated query goes: it needs query")
        hq = 0
    else:
        if inv_freq is None:
            raise KvCacheError("a query is there to be rotated: it needs inv_freq")
        if query.dim() != 3 or query.shape[0] != total or query.shape[2] != d:
            raise KvCacheError(f"query {tuple(query.shape)} does not match the keys' {tuple(key.shape)}")
        hq = query.shape[1]
    if inv_freq is not None and (inv_freq.dtype is not torch.float32 or inv_freq.shape != (d // 2,)
                                 or not inv_freq.is_contiguous()):
        raise KvCacheError(f"inv_freq must be a contiguous float32 tensor of {d // 2} elements")
    if out is not None and out.shape != query.shape:
        raise KvCacheError("out must match query's shape")
    for name, t in (("key", key), ("value", value), ("k_cache", k_cache), ("v_cache", v_cache), ("query", query),
                    ("out", out)):
        if t is None:
            continue
        if t.dtype is not dtype or t.device != dev:
            raise KvCacheError(f"{name} must share the cache's dtype and device")
        if t.stride(-1) != 1:
            raise KvCacheError(f"{name} must have a unit head_dim stride")
    if inv_freq is not None and inv_freq.device != dev:
        raise KvCacheError("inv_freq must be on the cache's device")
    if status is not None and (status.dtype is not torch.int32 or status.device != dev or status.numel() < 1):
        raise KvCacheError("status must be an int32 device tensor")
    if block_tables.dim() != 2:
        raise KvCacheError("block_tables must have two dimensions")
    num_seqs = block_tables.shape[0]
    if seq_lens.numel() != num_seqs or query_lens.numel() != num_seqs or query_start_loc.numel() != num_seqs + 1:
        raise KvCacheError("seq_lens/query_lens need num_seqs entries and query_start_loc num_seqs + 1")
    if dev.type != "cuda":
        raise KvCacheError("store_kv_hip needs device tensors")
    handle, on = _on(dev, stream)
    with on:
        if query is not None and out is None:
            out = torch.empty(query.shape, dtype=dtype, device=dev)
        if total == 0:
            return out
        bt = block_tables
        if bt.dtype is not torch.int32 or bt.device != dev or bt.stride(1) != 1:
            bt = _i32(bt, dev, "block_tables")
        sl, qsl, ql = (_i32(t, dev, n) for t, n in ((seq_lens, "seq_lens"), (query_start_loc, "query_start_loc"),
                                                    (query_lens, "query_lens")))
        qs, os_ = (query.stride(), out.stride()) if query is not None else ((0, 0), (0, 0))
        ks, vs, kc, vc = key.stride(), value.stride(), k_cache.stride(), v_cache.stride()
        a = NsKvStoreArgs(
            query.data_ptr() if query is not None else None, key.data_ptr(), value.data_ptr(), k_cache.data_ptr(),
            v_cache.data_ptr(), out.data_ptr() if query is not None else None,
            inv_freq.data_ptr() if inv_freq is not None else None, bt.data_ptr(), sl.data_ptr(), qsl.data_ptr(),
            ql.data_ptr(), status.data_ptr() if status is not None else None,
            qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], kc[0], kc[1], kc[2], vc[0], vc[1], vc[2], os_[0], os_[1],
            bt.stride(0), total, num_seqs, hq, hkv, d, bs, nb, bt.shape[1], _DTYPES[dtype])
        _check(lib.ns_kv_store(ctypes.byref(a), handle))
    return out


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
    the list.  One pool's calls run one after another; ``stream`` as in ``store_kv_hip``.
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
        pages, bs, heads, d = first.shape
        dev, slot = first.device, heads * d * first.element_size()
        if min(pages, bs) < 1 or slot < 16 or slot % 16 != 0:
            raise KvCacheError(f"a page's slot must be a positive multiple of 16 bytes (got {slot})")
        for name, t, shape in (("block_tables", block_tables, None), ("seq_lens", seq_lens, (block_tables.shape[0],)),
                               ("page_refs", page_refs, (pages,))):
            if t.dtype is not torch.int32 or t.device != dev or (shape is not None and t.shape != shape):
                raise KvCacheError(f"{name} must be an int32 tensor on the caches' device"
                                   + (f" of shape {shape}" if shape is not None else ""))
        if block_tables.dim() != 2 or block_tables.numel() == 0 or block_tables.stride(1) != 1 \
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
        _check(self._lib.ns_kv_scratch_bytes(block_tables.shape[0], pages, ctypes.byref(need)))
        self.k_caches, self.v_caches = list(k_caches), list(v_caches)
        self.block_tables, self.seq_lens, self.page_refs = block_tables, seq_lens, page_refs
        self.device, self.block_size, self.num_pages = dev, bs, pages
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._scratch = torch.zeros(int(need.value), dtype=torch.uint8, device=dev)
        self._tensors = torch.tensor([[c.data_ptr(), c.stride(0) * c.element_size()] for c in caches],
                                     dtype=torch.int64, device=dev)
        self._pool = NsKvPool(block_tables.data_ptr(), seq_lens.data_ptr(), page_refs.data_ptr(), self.status.data_ptr(),
                              self._tensors.data_ptr(), self._scratch.data_ptr(), int(need.value),
                              block_tables.stride(0), slot, block_tables.shape[0], block_tables.shape[1], pages,
                              len(caches), bs)
        self._ref = ctypes.byref(self._pool)

    @classmethod
    def empty(cls, k_caches, v_caches, max_seqs: int, max_pages_per_seq: int, reserved: int = 1):
        """A pool of no sequences over the caches.  The first ``reserved`` pages are never handed out (the reference
        keeps page 0 for padding)."""
        dev, pages = k_caches[0].device, k_caches[0].shape[0]
        refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        refs[:reserved] = 1
        return cls(k_caches, v_caches, torch.full((max_seqs, max_pages_per_seq), -1, dtype=torch.int32, device=dev),
                   torch.zeros(max_seqs, dtype=torch.int32, device=dev), refs)

    def _list(self, x, name):
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

    def extend(self, rows, lens, stream=None) -> None:
        """Row ``rows[i]`` grows to ``lens[i]`` tokens (its length grows with it) and gets the pages for them, the
        lowest free ones first.  A row is served if the pages that it and the rows listed before it ask for are all
        there; else it is left as it was (NO_PAGES).  At most MAX_ROWS rows a call."""
        handle, on = _on(self.device, stream)
        with on:
            rows, lens = self._two(rows, lens, ("rows", "lens"))
            _check(self._lib.ns_kv_extend(self._ref, rows.data_ptr(), lens.data_ptr(), rows.numel(), handle))

    def fork(self, parents, children, stream=None) -> None:
        """Row ``children[i]``, an empty one, becomes a copy of row ``parents[i]``: full pages are shared, the tokens
        of a last page that is not full are copied, in every layer, to a page of the child's own.  A child for which
        no page is left stays empty (NO_PAGES).  At most MAX_ROWS pairs, and no more than rows, a call."""
        handle, on = _on(self.device, stream)
        with on:
            parents, children = self._two(parents, children, ("parents", "children"))
            _check(self._lib.ns_kv_fork(self._ref, parents.data_ptr(), children.data_ptr(), parents.numel(), handle))

    def free(self, rows, stream=None) -> None:
        """The rows give up their pages and become empty; a page that no row names any more is free."""
        handle, on = _on(self.device, stream)
        with on:
            rows = self._list(rows, "rows")
            _check(self._lib.ns_kv_free(self._ref, rows.data_ptr(), rows.numel(), handle))

    def release(self, rows, window: int, sinks: int = 0, stream=None) -> None:
        """The rows give up the pages that no later token sees through ``window`` and ``sinks`` (those of
        ``paged_attention_hip``); their entries become -1."""
        if not 1 <= window < 2 ** 31:
            raise KvCacheError(f"window must be at least 1 and below 2^31 (got {window})")
        if not 0 <= sinks < 2 ** 31:
            raise KvCacheError(f"sinks must lie in [0, 2^31) (got {sinks})")
        handle, on = _on(self.device, stream)
        with on:
            rows = self._list(rows, "rows")
            _check(self._lib.ns_kv_release(self._ref, rows.data_ptr(), rows.numel(), window, sinks, handle))

    def copy(self, src, dst, into: Optional["PagePool"] = None, stream=None) -> None:
        """Pages ``src[i]`` to pages ``dst[i]``, in every layer, of this pool or of ``into``, a pool of pages alike.
        Within one pool no page is to be in ``dst`` twice or in both lists (checked for lists, not for tensors).
        Tables and counts stay as they are."""
        to = self if into is None else into
        self._alike(to)
        if to is self and not isinstance(src, torch.Tensor) and not isinstance(dst, torch.Tensor):
            src, dst = list(src), list(dst)
            if len(set(dst)) != len(dst) or set(src) & set(dst):
                raise KvCacheError("a page is named twice by dst, or by src and dst")
        handle, on = _on(self.device, stream)
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
        mine = {c.data_ptr() for c in self.k_caches + self.v_caches}
        if any(c.data_ptr() in mine for c in to.k_caches + to.v_caches):
            raise KvCacheError("the pools share a cache")
        return self._compact(to, stream)

    def _alike(self, to):
        if to is self:
            return
        a, b = self.k_caches[0], to.k_caches[0]
        if len(self.k_caches) != len(to.k_caches) or a.shape[1:] != b.shape[1:] or a.dtype is not b.dtype \
                or self.device != to.device:
            raise KvCacheError("the pools' caches differ in layers, page shape, dtype or device")

    def _compact(self, to, stream):
        handle, on = _on(self.device, stream)
        with on:
            page_map = torch.empty(self.num_pages, dtype=torch.int32, device=self.device)
            _check(self._lib.ns_kv_compact(self._ref, to._ref if to is not None else None, page_map.data_ptr(), handle))
        return page_map
