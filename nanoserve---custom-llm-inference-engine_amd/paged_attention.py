"""Paged attention on MI355X: the reference's kernel surface over the gfx950 HIP library.

``paged_attention_hip`` takes the arguments of the reference's
``paged_attention_triton`` (nanoserve/kernels/paged_attention_triton.py:134-170) and
``paged_attention_torch`` (nanoserve/kernels/paged_attention_torch.py:31-100) in the same order
with the same meaning, and returns a tensor shaped and typed like ``query``. The computation runs in
``libns_paged_attention.so`` (include/ns_paged_attention.h); there is no other path: a missing
library raises.

Differences from the reference's launcher, all on the host side:
  * decode batches (every ``query_lens`` entry 1, declared by ``max_query_len=1``): the
    per-query sequence index and KV position (paged_attention_triton.py:109-131) are found by
    the kernel itself from ``query_start_loc``, so no index tensors are built, and with
    ``max_seq_len`` given the call reads nothing on the host;
  * otherwise the batch layout (``seq_lens``, ``query_start_loc``, ``query_lens``) is read on the
    host once, as the reference's launcher reads ``seq_lens.tolist()`` and ``query_lens.tolist()``
    (paged_attention_triton.py:120-121, paged_attention_torch.py:51): sequences of at least
    ``PREFILL_MIN_QUERY`` query tokens (bfloat16 and float16) are cut into query tiles of
    ``128 // G`` tokens for the MFMA prefill kernel, which reads each key and value row once per
    tile; the other query tokens go to the per-token kernel.

``window`` and ``sinks``: attention with a sliding window and a few first tokens that stay visible
(the reference attends to the whole context).  The cache pages between the two are not read, so they
can be released (``kv_cache.PagePool.release``).
"""
from __future__ import annotations

import ctypes
import importlib
import os
from typing import Optional

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libns_paged_attention.so")

ABI_VERSION = 3
NS_PA_DTYPE_F32 = 0
NS_PA_DTYPE_BF16 = 1
NS_PA_DTYPE_F16 = 2
STATUS_BAD_BLOCK = 1
STATUS_SEQ_TOO_LONG = 2
STATUS_BAD_TILE = 4
TILE_COLUMNS = 128         # query columns of a prefill tile (NS_PA_TILE_COLUMNS): 128 // G tokens of G heads
PREFILL_MIN_QUERY = 2      # sequences with at least this many query tokens go by tile

EXPORTS = ("ns_pa_abi_version", "ns_pa_last_error", "ns_paged_attention_workspace_bytes",
           "ns_paged_attention_call_workspace", "ns_paged_attention", "ns_paged_attention_windowed_workspace",
           "ns_paged_attention_windowed")


class PagedAttentionError(RuntimeError):
    """An argument the library refused (the message is the library's)."""


class NsPagedAttnArgs(ctypes.Structure):
    """ns_paged_attn_args of include/ns_paged_attention.h, field for field."""

    _fields_ = [
        ("query", ctypes.c_void_p),
        ("k_cache", ctypes.c_void_p),
        ("v_cache", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("block_tables", ctypes.c_void_p),
        ("seq_lens", ctypes.c_void_p),
        ("query_start_loc", ctypes.c_void_p),
        ("query_lens", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_uint64),
        ("counters", ctypes.c_void_p),
        ("stride_q_token", ctypes.c_int64),
        ("stride_q_head", ctypes.c_int64),
        ("stride_k_block", ctypes.c_int64),
        ("stride_k_token", ctypes.c_int64),
        ("stride_k_head", ctypes.c_int64),
        ("stride_v_block", ctypes.c_int64),
        ("stride_v_token", ctypes.c_int64),
        ("stride_v_head", ctypes.c_int64),
        ("stride_o_token", ctypes.c_int64),
        ("stride_o_head", ctypes.c_int64),
        ("stride_bt_seq", ctypes.c_int64),
        ("total_q", ctypes.c_int32),
        ("num_seqs", ctypes.c_int32),
        ("num_heads_q", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("block_size", ctypes.c_int32),
        ("num_blocks", ctypes.c_int32),
        ("max_blocks_per_seq", ctypes.c_int32),
        ("max_seq_len", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("decode_tokens", ctypes.c_void_p),
        ("n_decode_tokens", ctypes.c_int32),
        ("prefill_tiles", ctypes.c_void_p),
        ("n_prefill_tiles", ctypes.c_int32),
    ]


_LIB: Optional[ctypes.CDLL] = None
_ATTEND = None    # the host module's function, and the addresses of the library's that it calls


def host_module(error):
    """The compiled host side of the attention's and the cache store's calls (csrc/ns_host.cpp)."""
    import torch  # noqa: F401  (its libraries are the module's)

    if not os.path.exists(os.path.join(HERE, "_ns_host.so")):
        raise error(f"{os.path.join(HERE, '_ns_host.so')} is not built (run __graft_entry__.build())")
    return importlib.import_module("._ns_host", __package__)


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load the HIP library (raises when it is not built: there is no fallback)."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not os.path.exists(path):
        raise PagedAttentionError(f"{path} is not built (run __graft_entry__.build())")
    lib = ctypes.CDLL(path)
    lib.ns_pa_abi_version.restype = ctypes.c_int
    lib.ns_pa_abi_version.argtypes = []
    lib.ns_pa_last_error.restype = ctypes.c_char_p
    lib.ns_pa_last_error.argtypes = []
    lib.ns_paged_attention_workspace_bytes.restype = ctypes.c_int
    lib.ns_paged_attention_workspace_bytes.argtypes = [ctypes.c_int32] * 5 + [ctypes.POINTER(ctypes.c_uint64)]
    lib.ns_paged_attention_call_workspace.restype = ctypes.c_int
    lib.ns_paged_attention_call_workspace.argtypes = [ctypes.POINTER(NsPagedAttnArgs),
                                                      ctypes.POINTER(ctypes.c_uint64),
                                                      ctypes.POINTER(ctypes.c_uint64)]
    lib.ns_paged_attention.restype = ctypes.c_int
    lib.ns_paged_attention.argtypes = [ctypes.POINTER(NsPagedAttnArgs), ctypes.c_void_p]
    lib.ns_paged_attention_windowed_workspace.restype = ctypes.c_int
    lib.ns_paged_attention_windowed_workspace.argtypes = [ctypes.POINTER(NsPagedAttnArgs), ctypes.c_int32,
                                                          ctypes.c_int32, ctypes.POINTER(ctypes.c_uint64),
                                                          ctypes.POINTER(ctypes.c_uint64)]
    lib.ns_paged_attention_windowed.restype = ctypes.c_int
    lib.ns_paged_attention_windowed.argtypes = [ctypes.POINTER(NsPagedAttnArgs), ctypes.c_int32, ctypes.c_int32,
                                                ctypes.c_void_p]
    if lib.ns_pa_abi_version() != ABI_VERSION:
        raise PagedAttentionError(f"ABI {lib.ns_pa_abi_version()} in {path}, expected {ABI_VERSION}")
    _LIB = lib
    return lib


def load_host() -> None:
    """The library and the host module that calls it."""
    global _ATTEND
    lib, host = load(), host_module(PagedAttentionError)
    host.set_errors(PagedAttentionError, None)
    _ATTEND = (host.attend, *(ctypes.cast(f, ctypes.c_void_p).value for f in (
        lib.ns_paged_attention_call_workspace, lib.ns_paged_attention, lib.ns_paged_attention_windowed_workspace,
        lib.ns_paged_attention_windowed, lib.ns_pa_last_error)))


def _check(rc: int) -> None:
    if rc != 0:
        raise PagedAttentionError(load().ns_pa_last_error().decode())


def workspace_bytes(total_q: int, num_heads_q: int, num_kv_heads: int, head_dim: int, max_seq_len: int) -> int:
    out = ctypes.c_uint64(0)
    _check(load().ns_paged_attention_workspace_bytes(total_q, num_heads_q, num_kv_heads, head_dim, max_seq_len,
                                                    ctypes.byref(out)))
    return int(out.value)


_COUNTERS = {}
_OUTGROWN = []    # counters that larger ones replaced: graphs captured on their stream before hold their addresses
_CAPTURED = {}    # by device and stream: a capture's id, and its counters


def _capture_id(handle):
    """The id of the capture that the stream of ``handle`` is in, or None."""
    state, number = ctypes.c_int(0), ctypes.c_ulonglong(0)
    info = load().hipStreamGetCaptureInfo   # of the HIP runtime that the library is linked with
    info.restype = ctypes.c_int
    info.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_ulonglong)]
    ok = info(handle, ctypes.byref(state), ctypes.byref(number)) == 0
    return int(number.value) if ok and state.value == 1 else None   # hipStreamCaptureStatusActive


def counters_for(device, n: int, stream=None):
    """A zero-filled int32 buffer of at least ``n`` arrival counters kept per device and stream
    (calls on one stream run one after another; calls on two streams may overlap, so they never
    share counters).  Every call leaves its counters at zero whatever its shape, so the buffer
    stays valid for all calls of its stream; it only grows, zero-filled on ``stream``, to at least twice its size,
    and what it replaces is kept for the graphs that hold it.  One made while ``stream`` is captured is filled by
    the graph, when it runs, so it serves the calls of that capture alone."""
    import torch

    dev = torch.device(device)
    s = stream if stream is not None else torch.cuda.current_stream(dev)
    key = (dev.index or 0, int(s.cuda_stream))
    buf = _COUNTERS.get(key)
    if buf is None or buf.numel() < n:
        with torch.cuda.stream(s):
            if torch.cuda.is_current_stream_capturing():
                number = _capture_id(int(s.cuda_stream))
                held = _CAPTURED.get(key)
                if held is None or held[0] != number or number is None or held[1].numel() < n:
                    held = _CAPTURED[key] = (number, torch.zeros(max(n, 1 << 12), dtype=torch.int32, device=dev))
                return held[1]
            if buf is not None:
                _OUTGROWN.append(buf)
                n = max(n, 2 * buf.numel())
            buf = torch.zeros(max(n, 1 << 16), dtype=torch.int32, device=dev)
        _COUNTERS[key] = buf
    return buf


def plan_tiles(seq_lens, query_start_loc, query_lens, num_heads_q: int, num_kv_heads: int):
    """Host plan of a batch with prefill chunks: (tiles, decode tokens) as int32 numpy arrays.
    Each sequence with at least PREFILL_MIN_QUERY query tokens is cut into tiles of
    TILE_COLUMNS // G consecutive tokens, (sequence, first token, count) each; every other query
    token is listed for the per-token kernel."""
    import numpy as np

    ql = np.asarray(query_lens, dtype=np.int64)
    qsl = np.asarray(query_start_loc, dtype=np.int64)
    bq = TILE_COLUMNS // (num_heads_q // num_kv_heads)
    tiles, tokens = [], []
    for s in range(ql.size):
        q, start = int(ql[s]), int(qsl[s])
        if q >= PREFILL_MIN_QUERY:
            for t in range(0, q, bq):
                tiles.append((s, start + t, min(bq, q - t)))
        elif q > 0:
            tokens.extend(range(start, start + q))
    return (np.asarray(tiles, dtype=np.int32).reshape(-1, 3), np.asarray(tokens, dtype=np.int32))


class PagedAttentionPlan:
    """The host plan of one batch layout, reusable by every layer's call of a step: the device
    lists of prefill tiles and per-token queries, and the layout's longest sequence and query.
    The reference's launcher reads the layout on every call (paged_attention_triton.py:120-121);
    with a plan the calls read nothing on the host."""

    def __init__(self, seq_lens, query_start_loc, query_lens, num_heads_q: int, num_kv_heads: int, device):
        import torch

        h_sl = np.asarray(seq_lens.cpu() if hasattr(seq_lens, "cpu") else seq_lens, dtype=np.int64).reshape(-1)
        h_qsl = np.asarray(query_start_loc.cpu() if hasattr(query_start_loc, "cpu") else query_start_loc,
                           dtype=np.int64).reshape(-1)
        h_ql = np.asarray(query_lens.cpu() if hasattr(query_lens, "cpu") else query_lens, dtype=np.int64).reshape(-1)
        self.num_heads_q, self.num_kv_heads = int(num_heads_q), int(num_kv_heads)
        self.total_q = int(h_ql.sum())
        self.max_seq_len = int(h_sl.max()) if h_sl.size else 0
        self.max_query_len = int(h_ql.max()) if h_ql.size else 0
        self.staged = None
        self.tokens = (0, 0)
        self.tiles = None
        if self.max_query_len >= PREFILL_MIN_QUERY:
            h_tiles, h_tokens = plan_tiles(h_sl, h_qsl, h_ql, num_heads_q, num_kv_heads)
            staged = torch.from_numpy(np.concatenate([h_tokens, h_tiles.reshape(-1)]).astype(np.int32))
            if torch.device(device).type == "cuda":
                staged = staged.pin_memory()
            self.staged = staged.to(device, non_blocking=True)
            # the per-token list starts the staged buffer (a valid address even when it is empty)
            self.tokens = (self.staged.data_ptr(), int(h_tokens.size))
            self.tiles = (self.staged.data_ptr() + 4 * int(h_tokens.size), int(h_tiles.shape[0]))


def paged_attention_hip(query, k_cache, v_cache, block_tables, seq_lens, query_start_loc, query_lens,
                        scale: float, block_size: int, *, max_seq_len: Optional[int] = None,
                        max_query_len: Optional[int] = None, plan: Optional[PagedAttentionPlan] = None,
                        window: Optional[int] = None, sinks: int = 0, out=None, workspace=None, counters=None,
                        status=None, stream=None):
    """Attention of every query token over its sequence's paged KV (the reference's
    ``paged_attention_triton``; same arguments, same result up to float32 rounding order).

    query (total_q, Hq, D); k_cache/v_cache (num_blocks, block_size, Hkv, D) of query's dtype;
    block_tables int (num_seqs, max_blocks_per_seq); seq_lens, query_lens int (num_seqs);
    query_start_loc int (num_seqs + 1). ``status``, if given, is an int32 device tensor of one
    element that the kernel ORs STATUS_* bits into (a block id outside the cache, a sequence longer
    than ``max_seq_len``): a caller that wants the check reads it after the call. ``workspace``
    (uint8, any contents) and ``counters`` (int32, zero-filled once; every call leaves it so) are
    allocated per call, resp. taken from this module's per-device, per-stream buffer, when not
    given.  ``out`` lies apart from the inputs.  ``max_query_len``: an upper bound of ``query_lens`` (1 for a decode step, which then
    takes the per-token kernel without reading the batch layout on the host).  ``plan``: a
    ``PagedAttentionPlan`` of this batch layout (then nothing is read on the host).  ``stream``: a
    ``torch.cuda.Stream`` or a raw HIP stream handle, default the current stream; the call's own temporaries
    are made on it, so nothing orders them against another.

    ``window`` (at least 1; None: the whole context): a query at KV position p sees the ``window`` positions up to
    its own, t > p - window, and the sequence's first ``sinks`` positions.  Block-table entries of blocks that no
    token of the call sees are not read, so they may hold anything (a released block's -1).  Query rows that are
    none of a sequence's ``query_lens`` tokens (a padded batch's) are left as they were.

    A call captured into a graph keeps the workspace and counters that it was captured with.  On a stream that made
    such a call before, these are the stream's counters: its graphs are then replayed one after another and not
    beside the stream's own calls, or given ``counters`` of their own.  On another each graph zero-fills counters of
    its own, once, for its calls.
    """
    import torch

    if _ATTEND is None:
        load_host()
    if window is not None and not 1 <= window < 2 ** 31:
        raise PagedAttentionError(f"window must be at least 1 and below 2^31 (got {window})")
    if not 0 <= sinks < 2 ** 31:
        raise PagedAttentionError(f"sinks must lie in [0, 2^31) (got {sinks})")
    index = query.get_device()
    if index < 0:
        raise PagedAttentionError("paged_attention_hip needs device tensors")
    if stream is None:
        if index == torch.cuda.current_device():   # already where the call goes: no stream to switch to and back
            return _paged_attention_on(index, torch._C._cuda_getCurrentRawStream(index), query, k_cache, v_cache,
                                       block_tables, seq_lens, query_start_loc, query_lens, scale, block_size,
                                       max_seq_len, max_query_len, plan, window, sinks, out, workspace, counters, status)
        s = torch.cuda.current_stream(query.device)
    elif isinstance(stream, torch.cuda.Stream):
        if stream.device_index != index:
            raise PagedAttentionError(f"the stream is one of device {stream.device_index}, the tensors are on device "
                                      f"{index}")
        s = stream
    elif int(stream) == 0:
        # the null stream is torch's default stream (an ExternalStream of handle 0 is not it)
        s = torch.cuda.default_stream(query.device)
    elif int(stream) == torch.cuda.current_stream(query.device).cuda_stream:
        s = torch.cuda.current_stream(query.device)
    else:
        s = torch.cuda.ExternalStream(int(stream), device=query.device)
    with torch.cuda.stream(s):
        return _paged_attention_on(index, s.cuda_stream, query, k_cache, v_cache, block_tables, seq_lens,
                                   query_start_loc, query_lens, scale, block_size, max_seq_len, max_query_len, plan,
                                   window, sinks, out, workspace, counters, status)


def _paged_attention_on(index, handle, query, k_cache, v_cache, block_tables, seq_lens, query_start_loc, query_lens,
                        scale, block_size, max_seq_len, max_query_len, plan, window, sinks, out, workspace, counters,
                        status):
    """paged_attention_hip with the stream of ``handle`` the current one: every temporary is made on it."""
    import torch

    attend, *entries = _ATTEND
    tokens = tiles = (0, 0)
    made = plan is None and query.dtype is not torch.float32 and (max_query_len is None
                                                                  or max_query_len >= PREFILL_MIN_QUERY)
    if made or plan is None and max_seq_len is None:
        # the batch layout is read on the host, once the call is known to be in order
        empty = attend(*entries, query, k_cache, v_cache, block_tables, seq_lens, query_start_loc, query_lens, scale,
                       block_size, 0, 0, 0, 0, 0, 0, 0, out, workspace, counters, status, False, -1)
        if query.shape[0] == 0:
            return empty
        if made:
            plan = PagedAttentionPlan(seq_lens, query_start_loc, query_lens, query.shape[1], k_cache.shape[2],
                                      query.device)
        else:
            max_seq_len = int(seq_lens.max().item()) if seq_lens.numel() else 0
    if plan is not None:
        # (a padded batch's rows behind the plan's are left alone with a window)
        total_q = query.shape[0]
        if not made and total_q > 0 and (plan.total_q > total_q or (window is None and plan.total_q < total_q)
                                         or plan.num_heads_q != query.shape[1] or plan.num_kv_heads != k_cache.shape[2]):
            raise PagedAttentionError("the plan was made for another batch layout or head layout")
        if max_seq_len is None:
            max_seq_len = plan.max_seq_len
        if plan.tiles is not None and query.dtype is not torch.float32:
            tokens, tiles = plan.tokens, plan.tiles
    own = counters is None
    if own:
        counters = _COUNTERS.get((index, handle))
    while True:
        got = attend(*entries, query, k_cache, v_cache, block_tables, seq_lens, query_start_loc, query_lens, scale,
                     block_size, max_seq_len, tokens[0], tokens[1], tiles[0], tiles[1], window or 0, sinks, out,
                     workspace, counters, status, own, handle)
        if type(got) is not int:
            return got
        counters = counters_for(query.device, got)


# the reference's name, so that nanoserve/model/attention.py:21 can import this module unchanged
paged_attention_triton = paged_attention_hip
