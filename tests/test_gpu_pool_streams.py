"""The page pool's tensors and the streams that its calls run on."""
import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu
KV = pkg("kv_cache")


def busy(stream):
    """Some milliseconds of work on ``stream``."""
    with torch.cuda.stream(stream):
        x = torch.randn(4096, 4096, device="cuda")
        for _ in range(40):
            x = x @ x * 0.01
    assert not stream.query()


def caches(device, n=1, pages=64):
    return [[torch.zeros(pages, 16, 2, 64, dtype=torch.bfloat16, device=device) for _ in range(n)] for _ in range(2)]


def test_a_new_pool_is_ready_on_any_stream(device):
    # made on a busy stream, used on another one at once: what its making fills is filled by then
    made, used = torch.cuda.Stream(device=device), torch.cuda.Stream(device=device)
    k, v = caches(device)
    torch.cuda.synchronize()
    busy(made)
    with torch.cuda.stream(made):
        pool = KV.PagePool.empty(k, v, 4, 8)
    assert made.query()
    with torch.cuda.stream(used):
        pool.extend([1, 9], [40, 1])
    torch.cuda.synchronize()
    assert pool.status.item() == KV.STATUS_BAD_ROW
    assert pool.seq_lens.tolist() == [0, 40, 0, 0] and pool.block_tables[1, :4].tolist() == [1, 2, 3, -1]


@pytest.mark.parametrize("way", ["current", "stream"])
@pytest.mark.parametrize("call", ["extend", "free", "copy", "compact", "into"])
def test_a_pool_dropped_while_a_stream_works_keeps_its_memory(device, call, way):
    side = torch.cuda.Stream(device=device)
    k, v = caches(device)
    pool = KV.PagePool.empty(k, v, 4, 8)
    other = KV.PagePool.empty(*caches(device), 4, 8)
    pool.extend([0, 1], [40, 17])
    rows, lens = (torch.tensor(x, dtype=torch.int32, device=device) for x in ([0, 1], [70, 33]))
    torch.cuda.synchronize()
    busy(side)
    with torch.cuda.stream(side if way == "current" else torch.cuda.current_stream()):
        kw = {} if way == "current" else {"stream": side}
        if call == "extend":
            pool.extend(rows, lens, **kw)
        elif call == "free":
            pool.free(rows, **kw)
        elif call == "copy":
            pool.copy(rows, lens, into=other, **kw)
        elif call == "compact":
            pool.compact(**kw)
        else:
            pool.compact_into(other, **kw)
    held = []
    for p in (pool, other) if call in ("copy", "into") else (pool,):
        held += [p.status, p._scratch, p._tensors, p.block_tables, p.seq_lens, p.page_refs, *p.k_caches, *p.v_caches]
    at = {t.data_ptr() for t in held}
    sizes = [t.numel() * t.element_size() for t in held]
    del pool, other, held, k, v, p
    assert not side.query()
    new = [torch.empty(n, dtype=torch.uint8, device=device) for n in sizes for _ in range(3)]
    assert not side.query()
    assert not at & {t.data_ptr() for t in new}
    side.synchronize()


def test_raw_handles_and_repeated_calls(device):
    side = torch.cuda.Stream(device=device)
    pool = KV.PagePool.empty(*caches(device), 4, 8)
    torch.cuda.synchronize()
    pool.extend([0], [20], stream=side.cuda_stream)
    assert side.cuda_stream not in pool._streams      # nothing is known of such a stream's life
    for n in (40, 41, 60):
        pool.extend([0], [n], stream=side)
    assert side.cuda_stream in pool._streams
    side.synchronize()
    assert pool.seq_lens.tolist() == [60, 0, 0, 0] and pool.status.item() == 0


def pool_over(k, v, device, tables=None, refs=None):
    pages = k.shape[0]
    tables = torch.full((4, 8), -1, dtype=torch.int32, device=device) if tables is None else tables
    refs = torch.zeros(pages, dtype=torch.int32, device=device) if refs is None else refs
    return KV.PagePool([k], [v], tables, torch.zeros(4, dtype=torch.int32, device=device), refs)


def test_compaction_into_memory_that_the_pools_share_is_refused(device):
    kv = torch.randn(100, 2, 16, 2, 64, device=device).to(torch.bfloat16)
    k, v = kv[:, 0], kv[:, 1]                      # interleaved: neighbours, but no byte in common
    whole = pool_over(k[:60], v[:60], device)
    for other in (pool_over(k[59:], v[59:], device), pool_over(k[40:61], v[70:91], device), pool_over(v[:60], k[:60], device)):
        with pytest.raises(KV.KvCacheError, match="share a cache"):
            whole.compact_into(other)
    tables = torch.full((7, 8), -1, dtype=torch.int32, device=device)
    refs = torch.zeros(100, dtype=torch.int32, device=device)
    low = pool_over(k[:60], v[:60], device, tables[:4], refs[:60])
    with pytest.raises(KV.KvCacheError, match="share a table"):
        low.compact_into(pool_over(k[60:], v[60:], device, tables[3:]))
    with pytest.raises(KV.KvCacheError, match="share a table"):
        low.compact_into(pool_over(k[60:], v[60:], device, refs=refs[56:96]))
    # the rest of the same tensors is another pool's to take
    want = kv.clone()
    low.extend([2, 0], [33, 20])                   # pages 0 .. 2 and 3, 4
    low.free([2])
    high = pool_over(k[60:], v[60:], device)
    page_map = low.compact_into(high)
    torch.cuda.synchronize()
    assert page_map[:6].tolist() == [-1, -1, -1, 0, 1, -1] and high.seq_lens.tolist() == [20, 0, 0, 0]
    assert high.block_tables[0, :3].tolist() == [0, 1, -1] and high.page_refs[:3].tolist() == [1, 1, 0]
    want[60:62] = want[3:5]
    assert torch.equal(kv, want)


def test_a_copy_into_another_pool_names_no_page_twice(device):
    pool, other = (pool_over(*(c[0] for c in caches(device)), device) for _ in range(2))
    pool.k_caches[0].normal_()
    for src in ([1, 2], torch.tensor([1, 2], dtype=torch.int32, device=device)):
        with pytest.raises(KV.KvCacheError, match="named twice"):
            pool.copy(src, [5, 5], into=other)
    pool.copy([1, 1], [5, 6], into=other)          # one page to two places
    pool.copy(iter([2, 3]), (3, 2), into=other)    # the numbers of two pools have nothing to do with each other
    torch.cuda.synchronize()
    at = [5, 6, 3, 2]
    assert torch.equal(other.k_caches[0][at], pool.k_caches[0][[1, 1, 2, 3]])
    assert torch.count_nonzero(other.k_caches[0]) == torch.count_nonzero(other.k_caches[0][at])
