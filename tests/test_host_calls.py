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
