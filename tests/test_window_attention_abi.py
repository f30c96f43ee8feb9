"""CPU checks of the windowed paged-attention entries: refusals, and workspaces that follow the window."""
import ctypes
import os

import numpy as np
import pytest

from conftest import pkg
from oracle import paged_attention_oracle as ORACLE

PA = pkg("paged_attention")


def built():
    if not os.path.exists(PA.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    return PA.load()


def args(**kw):
    a = PA.NsPagedAttnArgs()
    a.total_q, a.num_seqs, a.num_heads_q, a.num_kv_heads, a.head_dim = 4, 4, 24, 8, 128
    a.block_size, a.num_blocks, a.max_seq_len, a.dtype = 16, 4, 100000, PA.NS_PA_DTYPE_BF16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def workspace(a, window, sinks):
    b, c = ctypes.c_uint64(), ctypes.c_uint64()
    rc = PA.load().ns_paged_attention_windowed_workspace(ctypes.byref(a), window, sinks, ctypes.byref(b), ctypes.byref(c))
    return rc, int(b.value)


def test_refusals():
    lib = built()
    a = args()
    for window, sinks, word in ((0, 0, b"window"), (-5, 0, b"window"), (1, -1, b"sinks")):
        assert lib.ns_paged_attention_windowed(ctypes.byref(a), window, sinks, None) != 0
        assert word in lib.ns_pa_last_error()
        assert workspace(a, window, sinks)[0] != 0 and word in lib.ns_pa_last_error()
    assert lib.ns_paged_attention_windowed(None, 1, 0, None) != 0 and b"NULL" in lib.ns_pa_last_error()
    # the checks of the call without a window
    assert lib.ns_paged_attention_windowed(ctypes.byref(a), 8, 0, None) != 0 and b"NULL" in lib.ns_pa_last_error()
    assert workspace(args(num_kv_heads=7), 8, 0)[0] != 0
    assert lib.ns_paged_attention_windowed(ctypes.byref(args(total_q=0)), 8, 0, None) == 0   # nothing to do


@pytest.mark.parametrize("window,sinks,word", [(0, 0, "window"), (-1, 0, "window"), (2 ** 31, 0, "window"), (4, -1, "sinks"),
                                               (None, -1, "sinks"), (4, 2 ** 31, "sinks")])
def test_wrapper_refusals(window, sinks, word):
    built()
    import torch

    x = torch.zeros(1, 24, 128)
    with pytest.raises(PA.PagedAttentionError, match=word):
        PA.paged_attention_hip(x, x, x, x, x, x, x, 1.0, 16, window=window, sinks=sinks)


def test_workspace_follows_the_window():
    built()
    floats = 4 * 24 * (128 + 2) * 4      # a partition's partials, all rows and heads
    # 4 rows x 8 heads of 100,000 positions: partitions of at most 1024; of sinks and window alone: six even ones
    rc, whole = workspace(args(), 2 ** 31 - 1, 0)
    assert rc == 0 and whole % floats == 0 and -(-100000 // 1024) <= whole // floats <= -(-100000 // 512)
    rc, some = workspace(args(), 1000, 4)
    assert rc == 0 and some == floats * 6
    rc, none = workspace(args(), 33, 0)
    assert rc == 0 and none == 0         # one partition
    # sequences shorter than the window
    assert workspace(args(max_seq_len=640), 1000, 4) == (0, floats * 5)


def test_oracle_against_a_dense_mask():
    """The oracle's window and sinks against softmax over an explicitly masked score matrix."""
    rng = np.random.default_rng(1)
    n, m, d, bs, window, sinks = 41, 20, 8, 4, 7, 3
    blocks = -(-n // bs)
    perm = rng.permutation(blocks + 2)[:blocks]
    kc, vc = rng.standard_normal((2, blocks + 2, bs, 1, d))
    q = rng.standard_normal((m, 2, d))
    got = ORACLE.paged_attention(q, kc, vc, perm[None], [n], [0, m], [m], 0.3, bs, window=window, sinks=sinks)
    k, v = (x[perm].reshape(-1, d)[:n] for x in (kc, vc))
    for i in range(m):
        p = n - m + i
        for h in range(2):
            s = 0.3 * k @ q[i, h]
            for t in range(n):
                if t > p or (t <= p - window and t >= sinks):
                    s[t] = -np.inf
            w = np.exp(s - s.max())
            np.testing.assert_allclose(got[i, h], (w / w.sum()) @ v, rtol=1e-12, atol=1e-12)
