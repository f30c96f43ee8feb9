"""CPU checks of the host side of the attention's and the cache's calls (paged_attention.py, kv_cache.py,
csrc/ns_host.cpp): what it keeps, reads and holds around a launch."""
import contextlib
import types
import weakref

import pytest
import torch

from conftest import pkg

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
