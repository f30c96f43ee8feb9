"""Checks of the host side of the attention's and the cache's calls (paged_attention.py, kv_cache.py,
csrc/ns_host.cpp): what it keeps, reads and holds around a launch."""
import contextlib
import ctypes
import os
import random
import subprocess
import threading
import time
import types
import weakref

import pytest
import torch

from conftest import ROOT, pkg

KV = pkg("kv_cache")
PA = pkg("paged_attention")


@pytest.fixture
def host_stream(monkeypatch):
    """A stand-in for a stream whose counters live in host memory."""
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(PA, "_COUNTERS", {})
    return types.SimpleNamespace(cuda_stream=12345)


def test_counters_that_a_graph_may_hold_are_kept(host_stream):
    """A graph captured on the stream holds the address of the counters of its time: no later growth frees them."""
    first = PA.counters_for("cpu", 10, host_stream)
    assert PA.counters_for("cpu", first.numel(), host_stream) is first
    alive, total = [weakref.ref(first)], first.numel()
    n = first.numel()
    del first
    for _ in range(6):
        n += 1000
        now = PA.counters_for("cpu", n, host_stream)
        assert now.numel() >= n and not now.any()
        if alive[-1]() is not now:
            alive.append(weakref.ref(now))
            total += now.numel()
        n = now.numel()
        del now
    assert all(ref() is not None for ref in alive)
    assert total < 2 * n      # what is kept stays below what is in use


class Unread(torch.Tensor):
    """A tensor whose values the host does not ask for."""

    def max(self, *args, **kw):
        raise AssertionError("read on the host")

    item = tolist = cpu = numpy = max


@pytest.mark.parametrize("kw", [{}, {"max_query_len": 1}, {"max_seq_len": 8}, {"window": 5}])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_an_empty_query_reads_nothing_on_the_host(dtype, kw):
    PA.load_host()
    lens = torch.tensor([3, 4], dtype=torch.int32).as_subclass(Unread)
    zero = torch.zeros(2, dtype=torch.int32).as_subclass(Unread)
    starts = torch.zeros(3, dtype=torch.int32).as_subclass(Unread)
    q, cache = torch.empty(0, 8, 64, dtype=dtype), torch.empty(4, 16, 8, 64, dtype=dtype)
    out = torch.empty_like(q)
    args = dict(max_seq_len=None, max_query_len=None, plan=None, window=None, sinks=0, out=None, workspace=None,
                counters=None, status=None)
    args.update(kw)

    def call():
        return PA._paged_attention_on(0, 0, q, cache, cache, torch.zeros(2, 1, dtype=torch.int32), lens, starts, zero, 1.0,
                                      16, *args.values())

    got = call()
    assert got.shape == q.shape and got.dtype == dtype
    args["out"] = out
    assert call() is out


@pytest.fixture
def waiting(tmp_path):
    """Calls a function in a C library that returns once another Python thread has run meanwhile."""
    so = str(tmp_path / "wait_for_flag.so")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", os.path.join(ROOT, "tests", "native", "wait_for_flag.c"), "-o", so],
                   check=True)
    lib = ctypes.CDLL(so)
    entered, flag = (ctypes.c_int.in_dll(lib, n) for n in ("entered", "flag"))
    stop = threading.Event()

    def other():
        while not entered.value and not stop.is_set():
            time.sleep(0.001)
        flag.value = 1

    thread = threading.Thread(target=other)
    thread.start()
    yield tuple(ctypes.cast(f, ctypes.c_void_p).value for f in (lib.wait_for_flag, lib.no_flag))
    stop.set()
    thread.join()
    assert entered.value


def test_other_threads_run_during_an_attention_call(waiting):
    PA.load_host()
    attend, workspace = PA._ATTEND[:2]
    launch, why = waiting
    q, cache = torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(4, 16, 8, 64, dtype=torch.bfloat16)
    one = torch.ones(1, dtype=torch.int32)
    out = attend(workspace, launch, workspace, launch, why, q, cache, cache, torch.zeros(1, 1, dtype=torch.int32), one,
                 torch.tensor([0, 1], dtype=torch.int32), one, 1.0, 16, 1, 0, 0, 0, 0, 0, 0, None, None, None, None, True, 0)
    assert out.shape == q.shape


@pytest.mark.gpu
def test_other_threads_run_during_a_store(device, waiting):
    KV.load()
    x = torch.zeros(1, 8, 64, dtype=torch.bfloat16, device=device)
    cache = torch.zeros(4, 16, 8, 64, dtype=torch.bfloat16, device=device)
    one = torch.ones(1, dtype=torch.int32, device=device)
    starts = torch.tensor([0, 1], dtype=torch.int32, device=device)
    freq = torch.ones(32, device=device)
    out = KV._STORE[0](*waiting, x, x, cache, cache, one[None], one, starts, one, 16, x, freq, None, None, 0)
    assert out.shape == x.shape


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_other_threads_run_during_a_pool_call(device, waiting, kind):
    KV.load()
    rows = torch.zeros(1, dtype=torch.int32, device=device)
    launch, why = waiting
    assert KV._PAGES[0](kind, launch, why, 0, rows.get_device(), rows, rows, 8, 0, 0) is None


def bytes_of(t):
    """The addresses of a tensor's bytes."""
    at = torch.zeros(1, dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n)[None, :] * s).reshape(-1)
    return {t.data_ptr() + int(i) * t.element_size() + j for i in at for j in range(t.element_size())}


def overlap(a, b):
    return KV._overlap(KV._pieces(a), KV._pieces(b))


def test_overlap_of_pages_and_tables():
    """Against the sets of bytes themselves: slices, interleaved and strided pages, tables of one larger table."""
    rng = random.Random(5)
    room = torch.zeros(160, dtype=torch.int16)
    met = 0
    for _ in range(3000):
        pair = []
        for _ in range(2):
            n, page = rng.randint(1, 6), rng.choice((1, 2, 4, 7, 8))
            step = page + rng.choice((0, 0, 1, 4, 8, 9))
            last = (n - 1) * step + page
            pair.append(room[rng.randint(0, 159 - last):].as_strided((n, page), (step, 1), rng.randint(0, 159 - last)))
        want = bool(bytes_of(pair[0]) & bytes_of(pair[1]))
        met += want
        assert overlap(*pair) == overlap(*pair[::-1]) == want, [(t.data_ptr(), t.shape, t.stride()) for t in pair]
    assert 500 < met < 2500
    kv = torch.zeros(12, 2, 16, 2, 8)
    assert not overlap(kv[:, 0], kv[:, 1]) and not overlap(kv[:6, 0], kv[6:, 0])
    assert overlap(kv[:7, 0], kv[6:, 0]) and overlap(kv[:, 0], kv[3:4, 0]) and overlap(kv[:, 0], kv)
    assert not overlap(room[:0], room)


def test_overlap_of_pools_memory():
    rng = random.Random(6)
    room = torch.zeros(4096, dtype=torch.int16)
    met = 0
    for _ in range(400):
        caches, at = [], rng.randint(0, 3)
        for _ in range(8):     # beside each other, with gaps that the other pool's may fall into
            n, page = rng.randint(1, 4), rng.choice((8, 16))
            step = page + rng.choice((0, 8, 40))
            caches.append(room.as_strided((n, page), (step, 1), at))
            at += (n - 1) * step + page + rng.randint(0, 300)
        rng.shuffle(caches)
        a, b = KV._Memory(caches[:4], caches[:1]), KV._Memory([c[:, :8] for c in caches[4:]], caches[1:2])
        assert not a.shared_cache(b) and not b.shared_cache(a) and not a.shared_table(b)
        other = [room.as_strided((2, 8), (rng.choice((8, 16, 200)), 1), rng.randint(0, 3800)) for _ in range(3)]
        want = bool(set().union(*map(bytes_of, caches)) & set().union(*map(bytes_of, other)))
        met += want
        whole, part = KV._Memory(caches, caches), KV._Memory(other, other)
        assert whole.shared_cache(part) == part.shared_cache(whole) == want
        assert whole.shared_table(part) == any(overlap(x, y) for x, y in zip(caches, other))
    assert 40 < met < 360


class OnDevice(torch.Tensor):
    def get_device(self):
        return 0


def test_a_stream_of_another_device_is_refused(monkeypatch):
    class Stream:
        device_index, cuda_stream = 1, 4096

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(PA, "_paged_attention_on", lambda *a: pytest.fail("called"))
    x = torch.zeros(1, 8, 64).as_subclass(OnDevice)
    cache = torch.zeros(4, 16, 8, 64).as_subclass(OnDevice)
    n = torch.ones(1, dtype=torch.int32)
    with pytest.raises(PA.PagedAttentionError, match="device 1"):
        PA.paged_attention_hip(x, cache, cache, n[None], n, n, n, 1.0, 16, stream=Stream())
    with pytest.raises(KV.KvCacheError, match="device 1"):
        KV.store_kv_hip(x, x, cache, cache, n[None], n, n, n, 16, stream=Stream())
    with pytest.raises(KV.KvCacheError, match="device 1"):
        KV._on(0, Stream())
