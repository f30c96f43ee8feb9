"""GPU parity of windowed paged attention (sliding window and sinks) against the CPU oracle, with the
tolerances of the unwindowed kernels' suite (tests/pa_cases.py): half an ulp of the output type + K * u * cond."""
import ctypes
import math

import numpy as np
import pytest
import torch

from conftest import pkg
from pa_cases import assert_close_to_oracle, make_case, oracle_args, release_hidden, to_device
from oracle import paged_attention_oracle as PA

pytestmark = pytest.mark.gpu
A = pkg("paged_attention")


def run(case, device, window, sinks, **kw):
    c = to_device(case, device)
    print(f"window {window} sinks {sinks}: q {tuple(case['query'].shape)} {case['query'].dtype} seqs "
          f"{case['seq_lens'].tolist()} q_lens {case['query_lens'].tolist()}", flush=True)
    out = A.paged_attention_hip(c["query"], c["k_cache"], c["v_cache"], c["block_tables"], c["seq_lens"],
                                c["query_start_loc"], c["query_lens"], c["scale"], c["block_size"], window=window,
                                sinks=sinks, **kw)
    torch.cuda.synchronize()
    return out


def check(case, device, window, sinks, **kw):
    status = torch.zeros(1, dtype=torch.int32, device=device)
    out = run(case, device, window, sinks, status=status, **kw)
    ref = PA.paged_attention(**oracle_args(case), terms=True, window=window, sinks=sinks)
    assert_close_to_oracle(out, ref, case["query"].dtype)
    assert status.item() == 0
    return out


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (15, 4), (16, 16), (17, 37), (100, 0), (1024, 4), (5000, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_decode_rows(device, window, sinks, dtype):
    # lengths of one token to long ones around block and alignment edges, entries behind the window released
    case = make_case(1000 + window + sinks, [1, 2, 15, 16, 17, 33, 100, 513, 1040, 1500, 4000], [1] * 11, dtype=dtype)
    check(release_hidden(case, window, sinks), device, window, sinks)


@pytest.mark.parametrize("window,sinks", [(1, 0), (30, 5), (64, 0), (200, 70), (1000, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_prefill_chunks_and_decode_rows(device, window, sinks, dtype):
    case = make_case(1100 + window + sinks, [700, 300, 190, 1, 90, 45, 2300], [200, 300, 3, 1, 17, 1, 333], dtype=dtype)
    check(release_hidden(case, window, sinks), device, window, sinks)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 128), (16, 8, 64), (32, 8, 128), (32, 4, 64), (24, 8, 64), (64, 8, 128),
                                      (8, 8, 64), (16, 8, 128), (64, 8, 64)])
def test_head_layouts_and_dtypes(device, dtype, hq, hkv, d):
    case = make_case(1200 + hq + d, [70, 1, 460, 333, 600], [1, 1, 130, 333, 1], hq=hq, hkv=hkv, d=d, dtype=dtype)
    check(release_hidden(case, 77, 6), device, 77, 6)


@pytest.mark.parametrize("block_size", [1, 2, 4, 7, 8, 12, 32, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_block_sizes(device, block_size, dtype):
    # blocks smaller and larger than a load, the alignment and the window, powers of two and not
    case = make_case(1300 + block_size, [45, 230, 7, 1200, 301], [1, 30, 7, 1, 1], block_size=block_size, dtype=dtype,
                     d=64, hq=32)
    check(release_hidden(case, 50, 9), device, 50, 9)


def test_block_size_one_long_window(device):
    # blocks of one position: a partition's LDS list of blocks is as long as the partition
    case = make_case(1350, [9000] * 40, [1] * 40, hq=8, hkv=8, d=64, block_size=1)
    check(release_hidden(case, 6000, 1029), device, 6000, 1029)


@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31 - 1, 0), (600, 2 ** 31 - 1), (600, 600)])
def test_window_or_sinks_beyond_the_context(device, window, sinks):
    # everything visible: the function without a window
    case = make_case(1400, [513, 300, 600], [1, 300, 77])
    out = run(case, device, window, sinks)
    assert_close_to_oracle(out, PA.paged_attention(**oracle_args(case), terms=True), case["query"].dtype)


def poisoned(case, window, sinks, value):
    """K and V rows that no token of their sequence sees set to ``value`` (stored rows, and slots past the length)."""
    bs = case["block_size"]
    for s, (n, m) in enumerate(zip(case["seq_lens"].tolist(), case["query_lens"].tolist())):
        first = max(0, n - m - window + 1)
        for t in list(range(min(sinks, first), first)) + list(range(n, -(-n // bs) * bs)):
            b = int(case["block_tables"][s, t // bs])
            case["k_cache"][b, t % bs] = value
            case["v_cache"][b, t % bs] = value
    return case


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, "lowest"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_hidden_rows_hold_anything(device, value, dtype):
    value = torch.finfo(dtype).min if value == "lowest" else value
    plain = make_case(1500, [700, 90, 33, 1500], [1, 1, 20, 130], dtype=dtype)
    bad = make_case(1500, [700, 90, 33, 1500], [1, 1, 20, 130], dtype=dtype)
    want = run(plain, device, 60, 5)
    got = check(poisoned(bad, 60, 5, value), device, 60, 5)
    assert torch.equal(got, want)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", [(24, 8, 128), (8, 8, 64)])
def test_values_that_only_some_tokens_of_a_tile_see(device, value, dtype, hq, hkv, d):
    # an infinite or NaN element of one value row: it reaches the tokens that see the row, in that dim and KV head
    # only, and none before it or behind their window
    window, sinks, n, m = 40, 3, 400, 300
    case = make_case(1600, [n, 250], [m, 1], hq=hq, hkv=hkv, d=d, dtype=dtype)
    bs = case["block_size"]
    spots = [(0, 1, 2, 7), (0, 150, 3, 60), (0, 151, 3, 60), (0, 390, 0, 0), (1, 230, 5, 33)]   # row, t, head, dim
    for s, t, head, dim in spots:
        case["v_cache"][int(case["block_tables"][s, t // bs]), t % bs, head, dim] = value
    out = run(case, device, window, sinks).double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        ref = PA.paged_attention(**oracle_args(case), window=window, sinks=sinks)
    hit = np.zeros(out.shape, dtype=bool)
    g = hq // hkv
    for s, t, head, dim in spots:
        rows = range(m) if s == 0 else [m]
        for i in rows:
            p = n - m + i if s == 0 else 249
            if t <= p and (t > p - window or t < sinks):
                hit[i, head * g:(head + 1) * g, dim] = True
    assert hit.any() and not hit.all()
    clean = make_case(1600, [n, 250], [m, 1], hq=hq, hkv=hkv, d=d, dtype=dtype)
    for s, t, head, dim in spots:
        clean["v_cache"][int(clean["block_tables"][s, t // bs]), t % bs, head, dim] = 0.0
    clean_ref, cond = PA.paged_attention(**oracle_args(clean), terms=True, window=window, sinks=sinks)
    got = np.where(hit, 0.0, out)
    assert np.isfinite(got).all()
    assert_close_to_oracle(torch.from_numpy(got).to(dtype), (np.where(hit, 0.0, clean_ref), cond), dtype)
    if math.isnan(value):
        assert np.isnan(out[hit]).all()
    else:
        assert (out[hit] == value).all() and (ref[hit] == value).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tiles_in_parts(device, dtype):
    """One short chunk far into a context: its tile's steps are shared by several workgroups, whose partials are merged;
    with an infinite value in the first of them, and one in a row that the second half of the chunk alone sees."""
    n, m, window, sinks = 6000, 20, 4000, 5
    case = make_case(1650, [n], [m], hq=8, hkv=2, dtype=dtype)
    ref = PA.paged_attention(**oracle_args(case), terms=True, window=window, sinks=sinks)
    a = run(case, device, window, sinks)
    assert_close_to_oracle(a, ref, dtype)
    assert torch.equal(a, run(case, device, window, sinks))
    for t, dim in ((2, 9), (n - 8, 70)):
        case["v_cache"][int(case["block_tables"][0, t // 16]), t % 16, 1, dim] = math.inf
    got = run(case, device, window, sinks).double().cpu().numpy()
    hit = np.zeros(got.shape, dtype=bool)
    hit[:, 4:, 9] = True
    hit[m - 8:, 4:, 70] = True
    assert (got[hit] == math.inf).all() and np.isfinite(got[~hit]).all()
    assert_close_to_oracle(torch.from_numpy(np.where(hit, 0.0, got)).to(dtype), (np.where(hit, 0.0, ref[0]), ref[1]), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_nan_keys_and_queries_give_nan(device, dtype):
    # a NaN among the scores makes the token's whole output NaN, and no other's; in a chunk, in one partition and in many
    lens, qlens = [300, 200, 4000, 90], [100, 1, 1, 1]
    case = make_case(1660, lens, qlens, dtype=dtype)
    ref, cond = PA.paged_attention(**oracle_args(case), terms=True, window=50, sinks=2)
    wide, wide_cond = PA.paged_attention(**oracle_args(case), terms=True, window=3000, sinks=2)
    case["k_cache"][int(case["block_tables"][0, 270 // 16]), 270 % 16, 3, 7] = math.nan    # seen from position 270 on
    case["k_cache"][int(case["block_tables"][2, 3990 // 16]), 3990 % 16, 0, 7] = math.nan
    case["query"][10, 5] = math.nan
    case["query"][101, 23] = math.nan
    case["query"][102, 8] = math.nan
    for window, want, terms in ((50, ref, cond), (3000, wide, wide_cond)):
        got = run(case, device, window, 2).double().cpu().numpy()
        hit = np.zeros(got.shape, dtype=bool)
        hit[70:100, 9:12] = True
        hit[10, 5] = True
        hit[101, 23] = True
        hit[101, 0:3] = True      # sequence 2's token: its NaN key is KV head 0's
        hit[102, 8] = True
        assert np.isnan(got[hit]).all()
        assert_close_to_oracle(torch.from_numpy(np.where(hit, 0.0, got)).to(dtype), (np.where(hit, 0.0, want), terms), dtype)


def test_rows_that_are_no_tokens_are_left_alone(device):
    # a padded batch: rows behind the last sequence, and a sequence with fewer query tokens than its place holds
    case = make_case(1700, [300, 40, 500], [1, 1, 1])
    want = check(case, device, 64, 4)
    c = to_device(case, device)
    q = torch.randn(9, 24, 128, device=device).to(torch.bfloat16)
    place = [0, 3, 4]
    for i, at in enumerate(place):
        q[at] = c["query"][i]
    out = torch.full_like(q, 7.0)
    A.paged_attention_hip(q, c["k_cache"], c["v_cache"], c["block_tables"], c["seq_lens"],
                          torch.tensor([0, 3, 4, 9], dtype=torch.int32), c["query_lens"], c["scale"], c["block_size"],
                          window=64, sinks=4, max_query_len=1, max_seq_len=500, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out[place], want)
    rest = [i for i in range(9) if i not in place]
    assert (out[rest] == 7.0).all()
    # with prefill tiles beside them, from a plan of the batch without the padding
    case = make_case(1701, [300, 40], [30, 1])
    want = check(case, device, 20, 2)
    c = to_device(case, device)
    q = torch.cat([c["query"], c["query"][:5]])
    out = torch.full_like(q, 7.0)
    plan = A.PagedAttentionPlan(c["seq_lens"], c["query_start_loc"], c["query_lens"], 24, 8, device)
    A.paged_attention_hip(q, c["k_cache"], c["v_cache"], c["block_tables"], c["seq_lens"], c["query_start_loc"],
                          c["query_lens"], c["scale"], c["block_size"], window=20, sinks=2, plan=plan, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out[:31], want) and (out[31:] == 7.0).all()


def test_no_visible_key_gives_zeros(device):
    case = make_case(1750, [0, 20], [1, 1])
    out = check(case, device, 8, 2)
    assert torch.count_nonzero(out[0].float()).item() == 0
    # more query tokens than the sequence is long: the first of them see nothing
    case = make_case(1751, [5, 20], [9, 1])
    out = check(case, device, 3, 1)
    assert torch.count_nonzero(out[:4].float()).item() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_status_of_bad_blocks(device, dtype):
    # a visible block's bad entry is flagged and its keys skipped, a hidden one's is not looked at
    for lens, qlens in (([400, 400], [1, 1]), ([400, 400], [100, 30])):
        case = make_case(1800, lens, qlens, dtype=dtype)
        case["block_tables"][0, 24] = case["k_cache"].shape[0] + 3     # positions 384 .. 399 of row 0
        status = torch.zeros(1, dtype=torch.int32, device=device)
        out = run(case, device, 50, 4, status=status)
        assert status.item() == A.STATUS_BAD_BLOCK
        case["block_tables"][0, 24] = 0
        ref, cond = PA.paged_attention(**oracle_args(case), terms=True, window=50, sinks=4)
        keep = slice(qlens[0], None)
        assert_close_to_oracle(out[keep], (ref[keep], cond[keep]), dtype)
        skip = [i for i in range(qlens[0]) if lens[0] - qlens[0] + i < 384]   # tokens before those keys
        if skip:
            assert_close_to_oracle(out[skip], (ref[skip], cond[skip]), dtype)
    # the skipped keys weigh nothing: as if the sequence had ended before them
    case = make_case(1801, [384, 400], [1, 1], dtype=dtype)
    want = run(case, device, 50, 4)
    longer = make_case(1801, [384, 400], [1, 1], dtype=dtype)
    longer["seq_lens"][0] = 390
    longer["block_tables"][0, 24] = -5
    status.zero_()
    got = run(longer, device, 50 + 6, 4, status=status)
    assert status.item() == A.STATUS_BAD_BLOCK and torch.equal(got[0], want[0])   # row 1 sees six keys more


def test_long_contexts_stay_bounded(device):
    # a table of 60,000 blocks whose released entries are -1: the work and the workspace follow the window
    n, bs, window, sinks = 960_005, 16, 700, 4
    held = [0] + list(range((n - window) // bs, -(-n // bs)))
    case = make_case(1900, [len(held) * bs], [1], hq=32, hkv=8, d=128)
    bt = torch.full((1, -(-n // bs)), -1, dtype=torch.int32)
    bt[0, held] = case["block_tables"][0, :len(held)]
    case["block_tables"], case["seq_lens"] = bt, torch.tensor([n], dtype=torch.int32)
    check(case, device, window, sinks, max_query_len=1, max_seq_len=n)
    case["query"] = torch.randn(50, 32, 128).to(torch.bfloat16)
    case["query_lens"], case["query_start_loc"] = torch.tensor([50], dtype=torch.int32), torch.tensor([0, 50], dtype=torch.int32)
    check(case, device, window - 60, sinks)


def test_offsets_beyond_32_bits(device):
    # a cache of more than 2^32 elements, the blocks in use at its far end
    bs, hkv, d = 16, 8, 128
    blocks = 2 ** 32 // (bs * hkv * d) + 40
    case = make_case(1950, [300, 90], [1, 20], d=d)
    c = to_device(case, device)
    held = case["k_cache"].shape[0]
    big = [torch.empty((blocks, bs, hkv, d), dtype=torch.bfloat16, device=device) for _ in range(2)]
    for b, x in zip(big, (c["k_cache"], c["v_cache"])):
        b[-held:] = x
    out = A.paged_attention_hip(c["query"], big[0], big[1], c["block_tables"] + (blocks - held), c["seq_lens"],
                                c["query_start_loc"], c["query_lens"], c["scale"], bs, window=64, sinks=4)
    assert_close_to_oracle(out, PA.paged_attention(**oracle_args(case), terms=True, window=64, sinks=4), torch.bfloat16)


def test_strided_query_cache_and_output(device):
    case = make_case(2000, [50, 200, 90], [50, 1, 33], qkv_view=True)
    assert not case["query"].is_contiguous()
    check(case, device, 30, 4)
    # key and value rows interleaved in one tensor, an output with padded rows
    case = make_case(2001, [350, 200], [1, 77])
    c = to_device(case, device)
    both = torch.stack([c["k_cache"], c["v_cache"]], dim=2)      # (blocks, slots, 2, heads, dims)
    out = torch.zeros((78, 24, 160), dtype=torch.bfloat16, device=device)
    A.paged_attention_hip(c["query"], both[:, :, 0], both[:, :, 1], c["block_tables"], c["seq_lens"],
                          c["query_start_loc"], c["query_lens"], c["scale"], 16, window=30, sinks=4, out=out[:, :, :128])
    assert_close_to_oracle(out[:, :, :128], PA.paged_attention(**oracle_args(case), terms=True, window=30, sinks=4),
                           torch.bfloat16)
    assert (out[:, :, 128:] == 0).all()


def test_repeats_are_bit_equal_and_counters_end_at_zero(device):
    counters = torch.zeros(8192, dtype=torch.int32, device=device)
    ws = torch.full((384 << 20,), 0x7F, dtype=torch.uint8, device=device)   # the largest need: 342 MB
    for seed, lens, qlens in ((2100, [9000, 700, 5000], [1, 1, 1]), (2101, [4000, 700], [600, 1]), (2102, [3000] * 3, [1] * 3)):
        case = make_case(seed, lens, qlens)
        outs = [check(case, device, 2500, 4, workspace=ws, counters=counters) for _ in range(2)]
        assert torch.equal(outs[0], outs[1])
        assert torch.count_nonzero(counters).item() == 0


def test_captured_calls_and_side_streams(device):
    """Two captured steps over one cache, replayed several times among eager calls and on a side stream."""
    cases = [make_case(2200, [900, 300, 31], [1, 1, 1]), make_case(2201, [1200, 77], [1, 1])]
    dev = [to_device(c, device) for c in cases]
    want = [run(c, device, 256, 4) for c in cases]

    def call(c, **kw):
        return A.paged_attention_hip(c["query"], c["k_cache"], c["v_cache"], c["block_tables"], c["seq_lens"],
                                     c["query_start_loc"], c["query_lens"], c["scale"], c["block_size"], window=256,
                                     sinks=4, max_query_len=1, max_seq_len=int(c["block_tables"].shape[1]) * 16, **kw)

    ws = torch.empty(16 << 20, dtype=torch.uint8, device=device)
    counters = torch.zeros(4096, dtype=torch.int32, device=device)
    outs = [torch.zeros_like(c["query"]) for c in dev]
    graphs = []
    for c, out in zip(dev, outs):
        call(c, out=out, workspace=ws, counters=counters)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(c, out=out, workspace=ws, counters=counters)
        graphs.append(g)
    for _ in range(4):
        for out in outs:
            out.zero_()
        for g in graphs:
            g.replay()
        assert torch.equal(call(dev[0]), want[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    side = torch.cuda.Stream(device=device)
    torch.cuda.synchronize()
    got = call(dev[1], stream=side)
    raw = call(dev[1], stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want[1]) and torch.equal(raw, want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("window", [200, 420, 600, 1100, 1500, 2100, 3300, 4100, 7000])
def test_a_row_of_few_and_many_partitions(device, window, dtype):
    # one row: from one partition to more than two rounds of eight, with every remainder of the merge's loads
    case = make_case(2300 + window, [7300], [1], hq=8, hkv=2, d=64, dtype=dtype)
    check(release_hidden(case, window, 4), device, window, 4, max_query_len=1, max_seq_len=7300)


@pytest.mark.parametrize("window", [65000, 69000])
def test_more_partitions_than_a_wave_has_lanes(device, window):
    case = make_case(2400, [69500], [1], hq=4, hkv=1, d=64)
    check(release_hidden(case, window, 4), device, window, 4, max_query_len=1, max_seq_len=69500)


def needed(case, window, sinks, plan=None):
    """Bytes of workspace that a call is said to need."""
    a = A.NsPagedAttnArgs()
    a.total_q, a.num_heads_q, a.head_dim = case["query"].shape
    a.num_seqs, a.num_kv_heads, a.max_seq_len = len(case["seq_lens"]), case["k_cache"].shape[2], int(case["seq_lens"].max())
    a.dtype = A.NS_PA_DTYPE_BF16
    if plan is not None:
        a.decode_tokens, a.n_decode_tokens = plan.tokens
        a.prefill_tiles, a.n_prefill_tiles = plan.tiles
    n, counters = ctypes.c_uint64(), ctypes.c_uint64()
    assert A.load().ns_paged_attention_windowed_workspace(ctypes.byref(a), window, sinks, ctypes.byref(n),
                                                          ctypes.byref(counters)) == 0
    return int(n.value)


@pytest.mark.parametrize("lens,qlens", [([9000, 700, 5000], [1, 1, 1]), ([700, 9000, 4000, 3000], [300, 1, 17, 1]),
                                        ([2000, 2000], [600, 600])])
def test_a_workspace_of_the_size_asked_for(device, lens, qlens):
    """Split rows and tiles stay within it, and a listed row's place in the batch does not size it."""
    case = make_case(2500 + len(lens), lens, qlens)
    c = to_device(case, device)
    plan = A.PagedAttentionPlan(c["seq_lens"], c["query_start_loc"], c["query_lens"], 24, 8, c["query"].device)
    n = needed(case, 2500, 4, plan if plan.tiles is not None else None)
    assert n < 64 << 20
    room = torch.full((n + 4096,), 0x5A, dtype=torch.uint8, device=device)
    check(case, device, 2500, 4, plan=plan, workspace=room[:n])
    assert (room[n:] == 0x5A).all()
    if n > 0:
        with pytest.raises(A.PagedAttentionError, match="workspace"):
            run(case, device, 2500, 4, plan=plan, workspace=room[:n - 4])


@pytest.mark.parametrize("window", [None, 2500])
def test_graphs_of_a_new_stream_are_independent(device, window):
    """Counters first needed within a capture are the graph's: the second graph runs without the first."""
    cases = [make_case(2600, [3000, 2900], [1, 1]), make_case(2601, [2800, 3100], [1, 1])]
    dev = [to_device(c, device) for c in cases]
    kw = dict(max_query_len=1, max_seq_len=3100, window=window, sinks=0 if window is None else 4)

    def call(c, **more):
        return A.paged_attention_hip(c["query"], c["k_cache"], c["v_cache"], c["block_tables"], c["seq_lens"],
                                     c["query_start_loc"], c["query_lens"], c["scale"], c["block_size"], **kw, **more)

    want = [call(c) for c in dev]
    stream = torch.cuda.Stream(device=device)
    torch.cuda.synchronize()
    key = (stream.device.index or 0, stream.cuda_stream)
    A._COUNTERS.pop(key, None)   # handles come from a pool of streams
    graphs, outs = [], [torch.zeros_like(c["query"]) for c in dev]
    for c, out in zip(dev, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call(c, out=out)
            held = A._CAPTURED[key]
            out.zero_()
            call(c, out=out)     # the capture's second call takes the same counters
            assert A._CAPTURED[key] is held and (not graphs or held[1].data_ptr() != before)
        before = held[1].data_ptr()
        graphs.append(g)
    assert key not in A._COUNTERS
    for order in ((1, 0), (0, 1), (1, 1, 0)):
        for out in outs:
            out.zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert torch.equal(call(dev[0]), want[0])
