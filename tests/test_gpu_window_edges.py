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
