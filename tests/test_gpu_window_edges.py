"""Windowed attention where a chunk has more query tokens than its sequence is long, so that its first tokens stand
before the sequence's first position and see nothing: against the CPU oracle, with the bounds of tests/pa_cases.py."""
import math

import numpy as np
import pytest
import torch

from conftest import pkg
from pa_cases import assert_close_to_oracle, make_case, oracle_args, to_device
from oracle import paged_attention_oracle as PA

pytestmark = pytest.mark.gpu
A = pkg("paged_attention")


def run(case, device, window, sinks):
    c = to_device(case, device)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    print(f"window {window} sinks {sinks}: q {tuple(case['query'].shape)} {case['query'].dtype} seqs "
          f"{case['seq_lens'].tolist()} q_lens {case['query_lens'].tolist()}", flush=True)
    out = A.paged_attention_hip(c["query"], c["k_cache"], c["v_cache"], c["block_tables"], c["seq_lens"],
                                c["query_start_loc"], c["query_lens"], c["scale"], c["block_size"], window=window,
                                sinks=sinks, status=status)
    torch.cuda.synchronize()
    assert status.item() == 0
    return out


# one head a KV head: the four waves of a tile hold 32 tokens each, and a step that all of a wave's tokens have behind
# their windows is left out; three and eight heads: tiles of 42 and 16 tokens, the later ones with hidden positions
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 128), (8, 8, 64), (24, 8, 128), (64, 8, 64)])
@pytest.mark.parametrize("n,m,window,sinks", [(28, 128, 8, 0), (126, 128, 32, 0), (126, 128, 32, 3), (70, 300, 5, 1),
                                              (1, 40, 1, 0), (200, 333, 64, 20)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_more_query_tokens_than_positions(device, dtype, n, m, window, sinks, hq, hkv, d):
    case = make_case(3000 + n + m, [n, 90, 3], [m, 1, 5], hq=hq, hkv=hkv, d=d, dtype=dtype)
    out = run(case, device, window, sinks)
    assert_close_to_oracle(out, PA.paged_attention(**oracle_args(case), terms=True, window=window, sinks=sinks), dtype)
    assert torch.count_nonzero(out[:m - n].float()).item() == 0


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n,m,window,t", [(5, 9, 3, 2), (5, 9, 3, 4), (60, 100, 7, 50)])
@pytest.mark.parametrize("hq", [8, 24])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinite_values_there(device, dtype, hq, n, m, window, t, value):
    """One element of one value row, seen by ``window`` tokens at most: it reaches those, in its dim and KV head only."""
    head, dim, g = 2, 7, hq // 8
    case = make_case(3100 + n, [n], [m], hq=hq, hkv=8, dtype=dtype)
    at = (int(case["block_tables"][0, t // 16]), t % 16, head, dim)
    case["v_cache"][at] = 0.0
    ref, cond = PA.paged_attention(**oracle_args(case), terms=True, window=window, sinks=0)
    case["v_cache"][at] = value
    out = run(case, device, window, 0).double().cpu().numpy()
    hit = np.zeros(out.shape, dtype=bool)
    for i in range(m):
        if n - m + i - window < t <= n - m + i:
            hit[i, head * g:(head + 1) * g, dim] = True
    assert hit.any()
    got = np.where(hit, 0.0, out)
    assert np.isfinite(got).all()
    assert_close_to_oracle(torch.from_numpy(got).to(dtype), (np.where(hit, 0.0, ref), cond), dtype)
    assert (np.isnan(out[hit]) if math.isnan(value) else out[hit] == value).all()


@pytest.mark.parametrize("window", [None, 2500])
def test_a_graph_keeps_its_counters_when_the_stream_needs_more(device, window):
    """Captured on a stream that made an eager call before; then a call on that stream outgrows its counters."""
    case = make_case(3200, [3000, 2900], [1, 1])
    c = to_device(case, device)

    def call(out=None):
        return A.paged_attention_hip(c["query"], c["k_cache"], c["v_cache"], c["block_tables"], c["seq_lens"],
                                     c["query_start_loc"], c["query_lens"], c["scale"], c["block_size"], window=window,
                                     sinks=0 if window is None else 4, max_query_len=1, max_seq_len=3000, out=out)

    stream = torch.cuda.Stream(device=device)
    key = (stream.device.index or 0, stream.cuda_stream)
    A._COUNTERS.pop(key, None)   # handles come from a pool of streams
    with torch.cuda.stream(stream):
        want = call()
        held = A._COUNTERS[key]
        out = torch.zeros_like(c["query"])
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            call(out=out)
        assert A._COUNTERS[key] is held
        address, size = held.data_ptr(), held.numel()
        del held
        more = A.counters_for(device, size + 1, stream)
        assert more.numel() >= 2 * size and A._COUNTERS[key] is more
        # what is made now does not come to lie where the graph counts
        filled = [torch.full((size,), 7, dtype=torch.int32, device=device) for _ in range(8)]
        assert all(f.data_ptr() != address for f in filled)
        for _ in range(3):
            out.zero_()
            g.replay()
            assert torch.equal(call(), want)
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        assert all((f == 7).all() for f in filled) and not more.any()


@pytest.mark.parametrize("sink", [0.515625, 0.625])
@pytest.mark.parametrize("d", [64, 128])
def test_long_sums_of_equal_weights(device, d, sink):
    """2^20 keys alike but for sixteen sinks, whose values alone are not zero: equal weights, no power of two, are added
    one after another.  Rounding then errs to one side, an addition by at most 2^-24 of the sum so far, half of that on
    average over the additions of one whole sum: with one for each step of 64 positions 2^14 * 2^-25 = 2^-11 of the
    sum, besides the output's own 2^-11 and some 2^-20 for the weights.  (One for each pair of a lane's positions, 2^18,
    is off by 1.5 to 3.5 thousandths here.)"""
    bs, hkv, window, m = 16, 8, 2 ** 20, 8192
    n = window + m
    k = torch.full((2, bs, hkv, d), 0.5, dtype=torch.float16, device=device)
    k[1] = sink
    v = torch.zeros_like(k)
    v[1] = 32768.0
    q = torch.ones((m, hkv, d), dtype=torch.float16, device=device)
    tables = torch.zeros((1, n // bs), dtype=torch.int32, device=device)
    tables[0, 0] = 1
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)   # noqa: E731
    out = A.paged_attention_hip(q, k, v, tables, i32(n), i32(0, m), i32(m), d ** -0.5, bs, window=window, sinks=bs)
    w = bs * math.exp(d ** 0.5 * (sink - 0.5))
    want = 32768.0 * w / (w + window)
    off = (out.double().cpu() / want - 1.0).abs().max().item()
    print(f"d {d} sink {sink}: off by {off:.2e} of {want}", flush=True)
    assert off <= 2.0 ** -10 + 2.0 ** -20
