"""GPU parity of the paged cache's operators against the CPU oracle (oracle/kv_cache_oracle.py), and a decode loop of
all of them together.

Bound of a stored element that the rotation computes: half an ulp of the type + K * 2^-24 * (|x| + |y|) for the pair
(x, y).  K = 6: the angle's fraction of a turn is at most 1/2 and rounded once to float32 (2^-26 turns, 2 pi of them:
1.57 * 2^-24), sine and cosine are within 2 ulp (2 * 2^-24), a product and the sum round once each (2 * 2^-24)."""
import math

import numpy as np
import pytest
import torch

from conftest import pkg
from pa_cases import half_ulp, make_case
from oracle import kv_cache_oracle as ORACLE
from oracle import paged_attention_oracle as ATTENTION

pytestmark = pytest.mark.gpu
KV = pkg("kv_cache")
PA = pkg("paged_attention")


# ---------------------------------------------------------------------------------------------- store

def freqs(d, base=500000.0):
    return torch.tensor(base ** (-np.arange(0, d, 2) / d), dtype=torch.float32)


def new_rows(case, seed):
    """New keys and values for a case of make_case (whose caches hold other rows)."""
    g = torch.Generator().manual_seed(seed)
    total, hkv, d = case["query"].shape[0], case["k_cache"].shape[2], case["query"].shape[2]
    dt = case["query"].dtype
    return [torch.randn(total, hkv, d, generator=g).to(dt) for _ in range(2)]


def run_store(case, key, value, device, freq=None, rotate_query=True, **kw):
    x = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in case.items()}
    kc, vc = x["k_cache"].clone(), x["v_cache"].clone()
    if freq is not None:
        kw["inv_freq"] = freq.to(device)
        if rotate_query:
            kw.setdefault("query", x["query"])
            kw.setdefault("out", x["query"].clone())     # rows that are no token keep what is there
    print(f"store: q {tuple(case['query'].shape)} {case['query'].dtype} seqs {case['seq_lens'].tolist()} q_lens "
          f"{case['query_lens'].tolist()}", flush=True)
    out = KV.store_kv_hip(key.to(device), value.to(device), kc, vc, x["block_tables"], x["seq_lens"],
                          x["query_start_loc"], x["query_lens"], case["block_size"], **kw)
    torch.cuda.synchronize()
    return out, kc, vc


def close(got, want, scale, dtype):
    got = got.double().cpu().numpy()
    bound = np.where(scale > 0, half_ulp(np.maximum(np.abs(want), np.abs(got)), dtype) + 6 * 2.0 ** -24 * scale, 0.0)
    bad = np.abs(got - want) > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} elements off, the worst by {np.abs(got - want).max()}"


def check_store(case, device, freq=None, seed=1, rotate_query=True):
    key, value = new_rows(case, seed)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    out, kc, vc = run_store(case, key, value, device, freq, rotate_query, status=status)
    q, k, v, s_q, s_k = ORACLE.store(
        case["query"].double().numpy() if freq is not None and rotate_query else None, key.double().numpy(),
        value.double().numpy(), case["k_cache"].double().numpy(), case["v_cache"].double().numpy(),
        case["block_tables"].numpy(), case["seq_lens"].numpy(), case["query_start_loc"].numpy(),
        case["query_lens"].numpy(), case["block_size"], None if freq is None else freq.numpy())
    dt = case["query"].dtype
    close(kc, k, s_k, dt)
    assert np.array_equal(vc.double().cpu().numpy(), v)
    if q is not None:
        close(out, q, s_q, dt)
    else:
        assert out is None
    assert status.item() == 0
    return out, kc, vc


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", [(24, 8, 128), (32, 8, 64), (8, 8, 64), (64, 8, 128), (3, 1, 128), (16, 1, 64)])
def test_store_head_layouts_and_dtypes(device, dtype, hq, hkv, d):
    case = make_case(100 + hq + d, [1, 70, 260, 33, 16, 17], [1, 1, 30, 33, 0, 1], hq=hq, hkv=hkv, d=d, dtype=dtype)
    check_store(case, device, freqs(d))
    check_store(case, device)                                  # keys that come rotated
    check_store(case, device, freqs(d), rotate_query=False)    # keys alone


@pytest.mark.parametrize("block_size", [1, 7, 16, 24, 128])
def test_store_block_sizes(device, block_size):
    check_store(make_case(200 + block_size, [45, 130, 7], [1, 100, 7], block_size=block_size, hq=8, hkv=2), device, freqs(128))


@pytest.mark.parametrize("total", [4095, 4096, 4099])
def test_store_long_prompts(device, total):
    # around the number of tokens from which a workgroup takes several
    check_store(make_case(300 + total, [total + 900, 5], [total - 2, 2], hq=4, hkv=1, d=64), device, freqs(64))


def test_store_far_positions(device):
    # positions of millions: the angle is formed in 64 bits; only the page of the last token is in the tables
    for n in (1_000_003, 16_777_217, 40_000_000):
        case = make_case(400, [16], [5], hq=8, hkv=2, dtype=torch.float32)
        bt = torch.full((1, -(-n // 16)), -1, dtype=torch.int32)
        bt[0, (n - 5) // 16:] = torch.arange(1, 1 + bt.shape[1] - (n - 5) // 16, dtype=torch.int32)
        case["block_tables"], case["seq_lens"] = bt, torch.tensor([n], dtype=torch.int32)
        check_store(case, device, freqs(128))


def test_store_views_of_a_fused_projection_in_place(device):
    case = make_case(500, [50, 200], [50, 1])
    total, hq, hkv, d = 51, 24, 8, 128
    qkv = torch.randn(total, (hq + 2 * hkv) * d).to(torch.bfloat16)
    q, k, v = (t.view(total, -1, d) for t in qkv.split((hq * d, hkv * d, hkv * d), dim=1))
    x = {n: t.to(device) if isinstance(t, torch.Tensor) else t for n, t in case.items()}
    dev = qkv.to(device)
    dq, dk, dv = (t.view(total, -1, d) for t in dev.split((hq * d, hkv * d, hkv * d), dim=1))
    both = torch.stack([x["k_cache"], x["v_cache"]], dim=2)      # key and value rows interleaved
    out = KV.store_kv_hip(dk, dv, both[:, :, 0], both[:, :, 1], x["block_tables"], x["seq_lens"], x["query_start_loc"],
                          x["query_lens"], 16, query=dq, inv_freq=freqs(d).to(device), out=dq)
    assert out is dq
    wq, wk, wv, s_q, s_k = ORACLE.store(q.double().numpy(), k.double().numpy(), v.double().numpy(),
                                        case["k_cache"].double().numpy(), case["v_cache"].double().numpy(),
                                        case["block_tables"].numpy(), case["seq_lens"].numpy(),
                                        case["query_start_loc"].numpy(), case["query_lens"].numpy(), 16, freqs(d).numpy())
    close(dq, wq, s_q, torch.bfloat16)
    close(both[:, :, 0], wk, s_k, torch.bfloat16)
    assert np.array_equal(both[:, :, 1].double().cpu().numpy(), wv)
    assert torch.equal(dk.cpu(), k) and torch.equal(dv.cpu(), v)      # the inputs stay


def test_store_leaves_padding_and_bad_places_alone(device):
    case = make_case(600, [40, 3, 90], [2, 5, 3], hq=8, hkv=2, d=64)   # the second: more new tokens than its length
    key, value = new_rows(case, 2)
    want = check_store(case, device, freqs(64), seed=2)
    assert want is not None
    # rows behind the last sequence
    x = {n: t.to(device) if isinstance(t, torch.Tensor) else t for n, t in case.items()}
    pad = [torch.cat([t, torch.full_like(t[:3], 9.0)]).to(device) for t in (case["query"], key, value)]
    kc, vc, out = x["k_cache"].clone(), x["v_cache"].clone(), torch.full_like(pad[0], 7.0)
    KV.store_kv_hip(pad[1], pad[2], kc, vc, x["block_tables"], x["seq_lens"], x["query_start_loc"], x["query_lens"], 16,
                    query=pad[0], inv_freq=freqs(64).to(device), out=out)
    live = [0, 1, 4, 5, 6, 7, 8, 9]     # rows 2 and 3 are at positions -2 and -1
    assert torch.equal(out[live], want[0][live]) and (out[[2, 3, 10, 11, 12]] == 7.0).all()
    assert torch.equal(kc, want[1]) and torch.equal(vc, want[2])
    # a page outside the cache, and a position past the table
    for bad in ("entry", "columns"):
        y = dict(case)
        y["block_tables"] = case["block_tables"].clone()
        if bad == "entry":
            y["block_tables"][0, 2] = case["k_cache"].shape[0]
        else:
            y["block_tables"] = y["block_tables"][:, :2].contiguous()
        status = torch.zeros(1, dtype=torch.int32, device=device)
        out, kc, vc = run_store(y, key, value, device, freqs(64), status=status)
        assert status.item() == KV.STATUS_BAD_PAGE
        assert torch.equal(out[:2], want[0][:2])      # the query is rotated all the same
        q, k, v, s_q, s_k = ORACLE.store(None, key.double().numpy(), value.double().numpy(),
                                         case["k_cache"].double().numpy(), case["v_cache"].double().numpy(),
                                         y["block_tables"].numpy(), case["seq_lens"].numpy(),
                                         case["query_start_loc"].numpy(), case["query_lens"].numpy(), 16, freqs(64).numpy())
        close(kc, k, s_k, torch.bfloat16)
        assert np.array_equal(vc.double().cpu().numpy(), v)


def test_store_keeps_bits_of_values_and_special_keys(device):
    # values are copied bit for bit, infinities and NaN reach only their own pair
    case = make_case(700, [9], [9], hq=1, hkv=1, d=64)
    key, value = new_rows(case, 3)
    value.view(torch.int16)[:] = torch.arange(9 * 64, dtype=torch.int32).to(torch.int16).view(9, 1, 64) * 113
    key[4, 0, 5] = math.inf
    key[6, 0, 40] = math.nan
    out, kc, vc = run_store(case, key, value, device, freqs(64))
    got_v = vc[case["block_tables"][0, 0].item(), :9].cpu()
    assert torch.equal(got_v.view(torch.int16), value.view(torch.int16))
    got_k = kc[case["block_tables"][0, 0].item(), :9, 0].float().cpu()
    odd = ~torch.isfinite(got_k)
    want = torch.zeros_like(odd)
    want[4, [5, 37]] = True
    want[6, [8, 40]] = True
    assert torch.equal(odd, want)


def test_store_offsets_beyond_32_bits(device):
    bs, hkv, d = 16, 8, 128
    blocks = 2 ** 32 // (bs * hkv * d) + 40
    case = make_case(800, [300, 90], [1, 20])
    key, value = new_rows(case, 4)
    _, want_k, want_v = check_store(case, device, freqs(d), seed=4)
    held = case["k_cache"].shape[0]
    big = [torch.empty((blocks, bs, hkv, d), dtype=torch.bfloat16, device=device) for _ in range(2)]
    big[0][-held:], big[1][-held:] = case["k_cache"].to(device), case["v_cache"].to(device)
    KV.store_kv_hip(key.to(device), value.to(device), big[0], big[1], case["block_tables"].to(device) + (blocks - held),
                    case["seq_lens"], case["query_start_loc"], case["query_lens"], bs, inv_freq=freqs(d).to(device))
    assert torch.equal(big[0][-held:], want_k) and torch.equal(big[1][-held:], want_v)


def test_store_many_sequences(device):
    # more sequences than one round of the search holds, empty ones among them
    r = np.random.default_rng(9)
    q = r.integers(0, 3, 5000)
    case = make_case(900, q + r.integers(1, 40, 5000), q, hq=1, hkv=1, d=64)
    check_store(case, device, freqs(64))


# ---------------------------------------------------------------------------------------------- pages

class Both:
    """A pool on the device and the oracle's, driven alike.  Every page slot starts with a value of its own."""

    def __init__(self, device, rows, cols, pages, bs, layers=2, heads=1, d=8, dtype=torch.bfloat16, reserved=1, stride=1):
        g = torch.Generator().manual_seed(rows * 31 + pages)
        self.k, self.v = ([torch.randint(0, 2 ** 15, (pages * stride, bs, heads, d), generator=g, dtype=torch.int16)
                           .to(device).view(dtype)[::stride] for _ in range(layers)] for _ in range(2))
        self.pool = KV.PagePool.empty(self.k, self.v, rows, cols, reserved)
        self.bs, self.shape = bs, (rows, cols, pages)
        self.ref = ORACLE.Pool(self.pool.block_tables.cpu().numpy(), self.pool.seq_lens.cpu().numpy(),
                               self.pool.page_refs.cpu().numpy(), bs, self.contents(self.pool))

    @staticmethod
    def contents(pool):   # (page, slot, everything else)
        return torch.stack([c.view(torch.int16).cpu() for c in pool.k_caches + pool.v_caches], dim=2).numpy()

    def both(self, name, *args):
        print(name, [a if not hasattr(a, "__len__") or len(a) < 12 else len(a) for a in args], flush=True)
        got = getattr(self.pool, name)(*args)
        want = getattr(self.ref, name)(*args)
        return got, want

    def check(self, status=None):
        torch.cuda.synchronize()
        rows = np.arange(self.shape[0])
        assert np.array_equal(self.pool.seq_lens.cpu().numpy(), self.ref.lens)
        t = self.pool.block_tables.cpu().numpy()
        for r in rows:
            n = -(-int(self.ref.lens[r]) // self.bs)
            assert np.array_equal(t[r, :n], self.ref.tables[r, :n]), r
        assert np.array_equal(self.pool.page_refs.cpu().numpy(), self.ref.refs)
        used = self.ref.refs > 0
        assert np.array_equal(self.contents(self.pool)[used], self.ref.pages[used])
        assert self.pool.status.item() == (self.ref.status if status is None else status)
        # the counts are those of the tables, the reserved pages' aside
        count = np.bincount(t[t >= 0], minlength=self.shape[2])
        assert np.array_equal(count[1:], self.ref.refs[1:])


@pytest.mark.parametrize("bs,pages,layers", [(16, 300, 2), (1, 700, 1), (7, 200, 3), (32, 90, 5)])
def test_pool_against_the_oracle_over_random_calls(device, bs, pages, layers):
    b = Both(device, 24, 40, pages, bs, layers)
    r = np.random.default_rng(bs)
    for step in range(60):
        op = r.choice(["extend", "extend", "fork", "free", "release", "compact"])
        rows = r.permutation(24)[:r.integers(1, 9)].tolist()
        if op == "extend":
            lens = [int(b.ref.lens[x] + r.integers(0, 6 * bs)) for x in rows]
            b.both("extend", rows, lens)
        elif op == "fork":
            empty = [x for x in range(24) if b.ref.lens[x] == 0]
            n = min(len(empty), len(rows))
            b.both("fork", rows[:n], empty[:n])
        elif op == "free":
            b.both("free", rows)
        elif op == "release":
            b.both("release", rows, int(r.integers(1, 8 * bs)), int(r.integers(0, 3 * bs)))
        else:
            got, want = b.both("compact")
            assert np.array_equal(got.cpu().numpy(), want)
        b.check()


def test_pool_one_page_rows_and_lengths_of_zero(device):
    b = Both(device, 1, 1, 2, 16)
    b.both("extend", [0], [0])
    b.both("extend", [0], [1])
    b.check(0)
    b.both("extend", [0], [16])
    b.both("extend", [0], [17])      # past the table's columns
    b.check(KV.STATUS_BAD_LENGTH)
    b.both("free", [0])
    b.both("free", [0])
    b.both("free", [])
    b.both("extend", [], [])
    b.both("fork", [], [])
    b.check()


def test_pool_shortage_is_served_in_order(device):
    # rows are served while the pages that they and the rows before them ask for are there
    b = Both(device, 8, 20, 31, 4)
    b.both("extend", [5, 2, 7, 1, 0, 3], [40, 24, 60, 4, 0, 8])    # 10 + 6 + 15 = 31 > 30: row 7 and those after it wait
    assert b.ref.lens.tolist() == [0, 0, 24, 0, 0, 40, 0, 0]
    b.check(KV.STATUS_NO_PAGES)
    b.both("extend", [7, 1], [56, 4])       # 14 pages, the last: row 1 waits
    b.check(KV.STATUS_NO_PAGES)
    b.both("fork", [5, 5], [0, 4])          # full pages alone: nothing to hand out
    b.both("extend", [3], [1])
    b.check(KV.STATUS_NO_PAGES)
    b.both("free", [7])
    b.pool.status.zero_()
    b.ref.status = 0
    b.both("extend", [1], [30])
    b.both("fork", [1] * 3, [7, 3, 6])
    b.check(0)
    b.both("extend", [7, 3, 2], [32, 33, 27])    # in place, a page each for two of them: one is left
    b.check()


def test_pool_rows_listed_twice_or_not_there(device):
    b = Both(device, 6, 8, 60, 4)
    b.both("extend", [3, 0, 3, 9, -1, 0], [10, 3, 30, 4, 4, 32])   # the first listing counts
    b.check(KV.STATUS_BAD_ROW)
    b.both("fork", [3, 0, 3, 7, 3, 3], [1, 1, 3, 2, -4, 5])        # listed twice, not empty, no such parent or child
    b.check(KV.STATUS_BAD_ROW)
    b.both("fork", [2, 4], [4, 2])                                 # empty parents, children of one another
    b.check(KV.STATUS_BAD_ROW)
    b.both("extend", [0], [2])                                     # shorter than it is
    b.check(KV.STATUS_BAD_ROW | KV.STATUS_BAD_LENGTH)
    b.both("free", [3, 3, 6, 0, 3])
    b.both("release", [1, 1, -1], 3, 0)
    b.check()


def test_pool_many_samples_of_one_prompt(device):
    b = Both(device, 600, 30, 1200, 16)
    b.both("extend", [7], [16 * 29 + 5])
    b.both("fork", [7] * 599, [r for r in range(600) if r != 7])
    b.check(0)
    assert b.ref.refs.max() == 600
    b.both("extend", list(range(599, -1, -1)), [16 * 30] * 600)
    b.check(0)
    b.both("free", list(range(0, 600, 2)))
    b.both("compact")
    b.check(0)


@pytest.mark.parametrize("pages", [16384, 16385, 50001])
def test_pool_scans_many_pages(device, pages):
    # several rounds of the scan, the free pages at its end, in its middle and across rounds
    b = Both(device, 300, pages // 200 + 160, pages, 1, layers=1)
    b.both("extend", list(range(299)), [pages // 300] * 299)
    b.both("free", list(range(3, 299, 7)))
    b.both("extend", [299, 3, 10], [150, pages // 250, pages // 200])
    b.check(0)
    got, want = b.both("compact")
    assert np.array_equal(got.cpu().numpy(), want)
    b.check(0)
    b.both("extend", [17, 24], [70, pages // 200 + 2])
    b.check(0)


def test_pool_largest_lists(device):
    b = Both(device, 9000, 4, 30000, 2, layers=1)
    order = np.random.default_rng(2).permutation(9000).tolist()
    b.both("extend", order[:KV.MAX_ROWS], [1 + i % 6 for i in range(KV.MAX_ROWS)])
    b.check(0)
    b.both("free", order[:4000])
    b.both("fork", order[4000:8000], order[:4000])
    b.check(0)
    with pytest.raises(KV.KvCacheError, match="at most"):
        b.pool.extend(order, [1] * 9000)
    with pytest.raises(KV.KvCacheError, match="as many"):
        b.pool.extend([1, 2], [3])
    b.both("free", order)
    b.check(0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float8_e4m3fn])
def test_compact_into_another_pool(device, dtype):
    d = 16
    dt = torch.int16 if dtype is torch.bfloat16 else torch.int32 if dtype is torch.float32 else torch.int8
    g = torch.Generator().manual_seed(3)

    def caches(pages):
        return [torch.randint(-100, 100, (pages, 8, 2, d), generator=g, dtype=dt).to(device).view(dtype) for _ in range(6)]

    a, c = caches(90), caches(60)
    p = KV.PagePool.empty(a[:3], a[3:], 10, 9)
    p.extend(list(range(10)), [64] * 10)
    p.free([0, 2, 3, 7])
    p.fork([9, 9], [0, 2])
    p.extend([3], [57])
    p.release([1], 20, 9)
    small = KV.PagePool.empty(c[:3], c[3:], 10, 9)
    small.block_tables.fill_(5)
    before = [t.clone() for t in (p.block_tables, p.seq_lens, p.page_refs)] + [t.view(dt).clone() for t in a]
    ref = ORACLE.Pool(p.block_tables.cpu().numpy(), p.seq_lens.cpu().numpy(), p.page_refs.cpu().numpy(), 8,
                      torch.stack([t.view(dt).cpu() for t in a], dim=2).numpy())
    want = ref.compact()
    for _ in range(2):     # as often as one likes
        got = p.compact_into(small)
        torch.cuda.synchronize()
        assert np.array_equal(got.cpu().numpy(), want)
        m = int((ref.refs > 0).sum())
        assert m <= 60
        assert np.array_equal(small.page_refs.cpu().numpy(), ref.refs[:60])
        assert np.array_equal(small.seq_lens.cpu().numpy(), ref.lens)
        t = small.block_tables.cpu().numpy()
        for r in range(10):
            n = -(-int(ref.lens[r]) // 8)
            assert np.array_equal(t[r, :n], ref.tables[r, :n]) and (t[r, n:] == -1).all()
        now = torch.stack([x.view(dt).cpu() for x in c], dim=2).numpy()
        assert np.array_equal(now[:m], ref.pages[:m])
        after = [p.block_tables, p.seq_lens, p.page_refs] + [x.view(dt) for x in a]
        assert all(torch.equal(x, y) for x, y in zip(before, after))     # the source stays
    small.extend([4], [int(ref.lens[4]) + 1])     # a working pool
    assert small.status.item() == 0 and p.status.item() == 0
    # too small a pool is left alone
    tiny = caches(m - 1)
    q = KV.PagePool.empty(tiny[:3], tiny[3:], 10, 9)
    was = [x.view(dt).clone() for x in tiny] + [q.block_tables.clone(), q.page_refs.clone(), q.seq_lens.clone()]
    assert (p.compact_into(q) == -1).all() and p.status.item() == KV.STATUS_NO_PAGES
    assert all(torch.equal(x, y) for x, y in zip(was, [x.view(dt) for x in tiny] + [q.block_tables, q.page_refs, q.seq_lens]))
    with pytest.raises(KV.KvCacheError, match="another pool"):
        p.compact_into(p)
    with pytest.raises(KV.KvCacheError, match="share a cache"):
        p.compact_into(KV.PagePool.empty(a[3:], a[:3], 10, 9))
    with pytest.raises(KV.KvCacheError, match="differ"):
        p.compact_into(KV.PagePool.empty(c[:2], c[2:4], 10, 9))


def test_copy_of_pages(device):
    # pages with room between them, in a pool and into another one
    b = Both(device, 4, 4, 50, 16, layers=3, stride=3)
    src, dst = [3, 4, 7, 49], [10, 9, 8, 0]
    want = Both.contents(b.pool)
    b.pool.copy(src, dst)
    want[dst] = want[src]
    assert np.array_equal(Both.contents(b.pool), want)
    o = Both(device, 2, 2, 9, 16, layers=3)
    to = Both.contents(o.pool)
    b.pool.copy([40, 40, 1], [0, 8, 3], into=o.pool)
    to[[0, 8, 3]] = want[[40, 40, 1]]
    assert np.array_equal(Both.contents(o.pool), to) and np.array_equal(Both.contents(b.pool), want)
    assert b.pool.status.item() == 0
    b.pool.copy([1, 50, 2, -1], [30, 31, -7, 5])      # no such pages: the others are copied
    want[30] = want[1]
    assert b.pool.status.item() == KV.STATUS_BAD_PAGE and np.array_equal(Both.contents(b.pool), want)
    b.pool.copy([], [])
    for src, dst in (([1, 2], [3, 3]), ([1, 2], [2, 5])):
        with pytest.raises(KV.KvCacheError, match="named twice"):
            b.pool.copy(src, dst)
    with pytest.raises(KV.KvCacheError, match="differ"):
        b.pool.copy([1], [2], into=Both(device, 2, 2, 9, 8, layers=3).pool)


def test_pages_beyond_32_bits(device):
    # caches of 5 GB: pages at both ends, copied and compacted
    pages, bs = 40, 2 ** 20
    k = [torch.empty((pages, bs, 8, 8), dtype=torch.bfloat16, device=device) for _ in range(1)]
    v = [torch.empty((pages, bs, 8, 8), dtype=torch.bfloat16, device=device) for _ in range(1)]
    for t in k + v:
        for p in range(pages):
            t[p] = float(p)
    pool = KV.PagePool.empty(k, v, 3, pages)
    pool.extend([0, 1], [bs * 37, bs * 2 - 5])        # pages 1 .. 37, then 38 and 39
    pool.free([0])
    pool.fork([1], [2])                               # shares 38, copies 39 to 1
    assert pool.block_tables[:, :2].tolist() == [[-1, -1], [38, 39], [38, 1]]
    for t in k + v:
        assert (t[1, :bs - 5] == 39.0).all() and (t[1, bs - 5:] == 1.0).all()
    pool.compact()                                    # 38 and 39 to 2 and 3
    assert pool.block_tables[:, :2].tolist() == [[-1, -1], [2, 3], [2, 1]]
    for t in k + v:
        assert (t[2] == 38.0).all() and (t[3] == 39.0).all() and (t[1, :bs - 5] == 39.0).all()
    assert pool.status.item() == 0


def test_pool_captured_and_on_side_streams(device):
    b = Both(device, 12, 10, 200, 4, layers=2)
    b.both("extend", list(range(8)), [30, 7, 16, 33, 1, 12, 39, 20])
    rows = torch.tensor([8, 9, 10], dtype=torch.int32, device=device)
    parents = torch.tensor([0, 3, 6], dtype=torch.int32, device=device)
    lens = torch.tensor([37, 40, 40], dtype=torch.int32, device=device)

    def step(pool, **kw):
        pool.free(rows, **kw)
        pool.fork(parents, rows, **kw)
        pool.extend(rows, lens, **kw)
        pool.release(rows, 9, 3, **kw)

    step(b.pool)
    torch.cuda.synchronize()
    for name, args in (("fork", (parents, rows)), ("extend", (rows, lens)), ("release", (rows, 9, 3))):
        getattr(b.ref, name)(*[a.tolist() if isinstance(a, torch.Tensor) else a for a in args])
    b.check(0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(b.pool)
    for _ in range(4):      # free, then the same again: every replay ends where the first one did
        g.replay()
        b.check(0)
    side = torch.cuda.Stream(device=device)
    torch.cuda.synchronize()
    step(b.pool, stream=side)
    step(b.pool, stream=side.cuda_stream)
    side.synchronize()
    b.check(0)
    step(b.pool, stream=0)
    torch.cuda.default_stream(device).synchronize()
    b.check(0)


# ----------------------------------------------------------------------------------------- all together

def rotated(x, pos, freq):
    a = pos[:, None, None] * freq[None, None, :]
    lo, hi = np.split(x, 2, axis=-1)
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], axis=-1)


@pytest.mark.parametrize("dtype,captured", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_a_serving_loop_over_a_bounded_cache(device, dtype, captured):
    """Prompts in chunks, samples forked from them, decode steps far past what the cache could hold, a compaction in
    between: every attention output against attention over all rows that were ever stored, kept on the host."""
    hq, hkv, d, bs, window, sinks, rows = 8, 2, 64, 4, 21, 3, 6
    pages = 80
    k, v = (torch.zeros((pages, bs, hkv, d), dtype=dtype, device=device) for _ in range(2))
    pool = KV.PagePool.empty([k], [v], rows, 300)
    freq = freqs(d).to(device)
    g = torch.Generator().manual_seed(5)
    held = {r: ([], []) for r in range(rows)}      # every row's keys (rotated, rounded) and values so far
    status = torch.zeros(1, dtype=torch.int32, device=device)

    def fresh(n):
        return [torch.randn(n, h, d, generator=g).to(dtype).to(device) for h in (hq, hkv, hkv)]

    def attend(x, at, lens, qlens, **known):
        qsl = torch.tensor(np.concatenate([[0], np.cumsum(qlens)]), dtype=torch.int32, device=device)
        ql = torch.tensor(qlens, dtype=torch.int32, device=device)
        tables, sl = pool.block_tables[at].contiguous(), pool.seq_lens[at].contiguous()
        q = KV.store_kv_hip(x[1], x[2], k, v, tables, sl, qsl, ql, bs, query=x[0], inv_freq=freq, status=status)
        out = PA.paged_attention_hip(q, k, v, tables, sl, qsl, ql, d ** -0.5, bs, window=window, sinks=sinks,
                                     status=status, **known)
        return q, out

    def check(x, q, out, at, lens, qlens):
        torch.cuda.synchronize()
        i = 0
        for r, n, m in zip(at, lens, qlens):
            pos = np.arange(n - m, n)
            new = torch.from_numpy(rotated(x[1][i:i + m].double().cpu().numpy(), pos, freq.double().cpu().numpy())).to(dtype)
            for j in range(m):
                held[r][0].append(new[j].double().numpy())
                held[r][1].append(x[2][i + j].double().cpu().numpy())
            kc, vc = (np.stack(t)[None] for t in held[r])
            ref, cond = ATTENTION.paged_attention(q[i:i + m].double().cpu().numpy(), kc, vc, np.zeros((1, 1), dtype=int),
                                                  [n], [0, m], [m], d ** -0.5, n, terms=True, window=window, sinks=sinks)
            got = out[i:i + m].double().cpu().numpy()
            # a stored key may round to its neighbour where the rotation's float32 lies near the middle of two: one
            # ulp of one element moves the output by no more than 2^-7 (bfloat16), 2^-23 (float32) of the condition
            tol = half_ulp(np.maximum(np.abs(ref), np.abs(got)), dtype) + (2.0 ** -7 if dtype is torch.bfloat16 else 2.0 ** -18) * cond
            assert (np.abs(got - ref) <= tol).all(), (r, n, float((np.abs(got - ref) / tol).max()))
            i += m

    # two prompts of 50 and 33 tokens, in chunks
    for at, lens, qlens in (([0, 1], [30, 33], [30, 33]), ([0], [50], [20])):
        x = fresh(sum(qlens))
        pool.extend(at, lens)
        check(x, *attend(x, at, lens, qlens), at, lens, qlens)
    pool.release([0, 1], window, sinks)
    # two samples of the first, one of the second
    pool.fork([0, 0, 1], [2, 3, 4])
    for c, p in ((2, 0), (3, 0), (4, 1)):
        held[c] = (list(held[p][0]), list(held[p][1]))
    at = [0, 1, 2, 3, 4]
    lens = [50, 33, 50, 50, 33]
    at_dev = torch.tensor(at, dtype=torch.int32, device=device)
    one = torch.ones(5, dtype=torch.int32, device=device)
    qsl = torch.arange(6, dtype=torch.int32, device=device)
    x = fresh(5)
    q_out, out = torch.empty_like(x[0]), torch.empty_like(x[0])
    now = torch.tensor(lens, dtype=torch.int32, device=device)
    ws, counters = torch.empty(1 << 20, dtype=torch.uint8, device=device), torch.zeros(256, dtype=torch.int32, device=device)

    def step():
        now.add_(one)
        pool.extend(at_dev, now)
        KV.store_kv_hip(x[1], x[2], k, v, pool.block_tables[:5], pool.seq_lens[:5], qsl, one, bs, query=x[0],
                        inv_freq=freq, out=q_out, status=status)
        PA.paged_attention_hip(q_out, k, v, pool.block_tables[:5], pool.seq_lens[:5], qsl, one, d ** -0.5, bs,
                               max_query_len=1, max_seq_len=1200, window=window, sinks=sinks, out=out, workspace=ws,
                               counters=counters, status=status)
        pool.release(at_dev, window, sinks)

    graph = None
    for i in range(130):       # 5 rows of up to 180 tokens through 79 pages of 4
        for dst, src in zip(x, fresh(5)):
            dst.copy_(src)
        if captured and i == 3:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        if graph is None:
            step()
        else:
            graph.replay()
        lens = [n + 1 for n in lens]
        check(x, q_out, out, at, lens, [1] * 5)
        if i == 60:
            pool.compact()
    assert pool.status.item() == 0 and status.item() == 0
    assert pool.seq_lens[:5].tolist() == lens
    used = int((pool.page_refs > 0).sum())
    assert used <= 1 + 5 * ((window + bs - 1) // bs + 2)
    pool.free(at)
    assert int((pool.page_refs > 0).sum()) == 1
