"""CPU checks of the paged-cache library: exports, struct layouts, scratch sizes, and refusals before any launch."""
import ctypes
import os
import re
import subprocess
import tempfile

import numpy as np
import pytest
import torch

from conftest import ROOT, pkg
from oracle import kv_cache_oracle as ORACLE

KV = pkg("kv_cache")
HEADER = os.path.join(ROOT, "include", "ns_kv_cache.h")


def built():
    if not os.path.exists(KV.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    return KV.load()


def test_exports_and_version():
    txt = open(HEADER).read()
    names = sorted(set(re.findall(r"^\s*(?:int|const char\*)\s+(ns_\w+)\s*\(", txt, flags=re.M)))
    assert names == sorted(KV.EXPORTS)
    lib = built()
    for name in names:
        assert hasattr(lib, name), name
    assert lib.ns_kv_abi_version() == KV.ABI_VERSION == int(re.search(r"#define NS_KV_ABI_VERSION (\d+)", txt).group(1))
    assert KV.MAX_ROWS == int(re.search(r"#define NS_KV_MAX_ROWS (\d+)", txt).group(1))
    for name in ("BAD_PAGE", "NO_PAGES", "BAD_ROW", "BAD_LENGTH"):
        assert getattr(KV, "STATUS_" + name) == int(re.search(rf"#define NS_KV_STATUS_{name} (\d+)", txt).group(1))


@pytest.mark.parametrize("struct,cls", [("ns_kv_store_args", KV.NsKvStoreArgs), ("ns_kv_pool", KV.NsKvPool)])
def test_struct_layout_matches_header(struct, cls):
    txt = open(HEADER).read()
    body = txt[txt.index(f"typedef struct {struct}"):txt.index(f"}} {struct};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for decl in re.findall(r"^\s*([^/{}]+?);", body, flags=re.M):
        names += [n.strip().lstrip("*") for n in re.sub(r"^.*?\b(\w+)\s*(,|$)", r"\1\2", decl, count=1).split(",")]
    assert names == [f[0] for f in cls._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"ns_kv_cache.h\"\nint main(void) {\n"
    src += f'  printf("%zu\\n", sizeof({struct}));\n'
    src += "".join(f'  printf("%zu\\n", offsetof({struct}, {n}));\n' for n in names) + "  return 0;\n}\n"
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        with open(c, "w") as f:
            f.write(src)
        rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
        subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", "-I", os.path.dirname(HEADER), "-I",
                        os.path.join(rocm, "include"), c, "-o", exe], check=True)
        got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, n).offset for n in names]


def store_args(**kw):
    a = KV.NsKvStoreArgs()
    a.total, a.num_seqs, a.num_heads_q, a.num_kv_heads, a.head_dim = 4, 2, 24, 8, 128
    a.block_size, a.num_blocks, a.max_blocks_per_seq, a.dtype = 16, 4, 2, KV.NS_KV_DTYPE_BF16
    for n in ("key", "value", "k_cache", "v_cache", "block_tables", "seq_lens", "query_start_loc", "query_lens"):
        setattr(a, n, 4096)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=7), "dtype"), (dict(head_dim=96), "head_dim"), (dict(total=-1), "total"), (dict(num_kv_heads=0), "num_kv_heads"),
    (dict(query=4096, out=4096), "inv_freq"), (dict(out=4096), "come together"),
    (dict(query=4096, inv_freq=4096), "come together"), (dict(query=4096, inv_freq=4096, out=4096, num_heads_q=0), "num_heads_q"),
    (dict(num_seqs=0), "num_seqs"), (dict(block_size=0), "block_size"), (dict(num_blocks=0), "num_blocks"),
    (dict(max_blocks_per_seq=-1), "max_blocks"), (dict(key=None), "NULL"), (dict(query_lens=None), "NULL"),
    (dict(stride_k_token=4), "16 bytes"), (dict(stride_k_block=-8), "16 bytes"), (dict(value=4100), "aligned")])
def test_store_refusals(kw, word):
    lib = built()
    assert lib.ns_kv_store(ctypes.byref(store_args(**kw)), None) != 0
    assert word in lib.ns_kv_last_error().decode()


def test_an_empty_store_is_a_no_op():
    assert built().ns_kv_store(ctypes.byref(store_args(total=0)), None) == 0
    assert built().ns_kv_store(None, None) != 0


def pool(**kw):
    p = KV.NsKvPool()
    for n in ("block_tables", "seq_lens", "page_refs", "tensors", "scratch"):
        setattr(p, n, 4096)
    p.scratch_bytes, p.stride_bt_row, p.slot_bytes = 1 << 20, 8, 2048
    p.num_rows, p.num_cols, p.num_pages, p.num_tensors, p.block_size = 4, 8, 64, 2, 16
    for n, v in kw.items():
        setattr(p, n, v)
    return p


@pytest.mark.parametrize("kw,word", [
    (dict(num_rows=0), "needs rows"), (dict(num_pages=0), "needs rows"), (dict(block_size=0), "block size"),
    (dict(page_refs=None), "NULL"), (dict(scratch=None), "NULL"), (dict(stride_bt_row=7), "stride_bt_row"),
    (dict(slot_bytes=24), "slot_bytes"), (dict(slot_bytes=0), "slot_bytes"), (dict(page_refs=4100), "aligned"),
    (dict(scratch_bytes=16), "scratch of"), (dict(num_tensors=70000), "tensors")])
def test_pool_refusals(kw, word):
    lib = built()
    p = ctypes.byref(pool(**kw))
    for rc in (lambda: lib.ns_kv_extend(p, 4096, 4096, 1, None), lambda: lib.ns_kv_fork(p, 4096, 4096, 1, None),
               lambda: lib.ns_kv_free(p, 4096, 1, None), lambda: lib.ns_kv_release(p, 4096, 1, 8, 0, None),
               lambda: lib.ns_kv_copy(p, p, 4096, 4096, 1, None), lambda: lib.ns_kv_compact(p, None, 4096, None)):
        assert rc() != 0
        assert word in lib.ns_kv_last_error().decode()


def test_list_refusals_and_empty_lists():
    lib = built()
    good = pool()
    p = ctypes.byref(good)

    def refused(rc, word):
        assert rc != 0 and word in lib.ns_kv_last_error().decode(), lib.ns_kv_last_error()

    refused(lib.ns_kv_extend(p, 4096, None, 1, None), "NULL")
    refused(lib.ns_kv_extend(p, 4096, 4096, -1, None), "length")
    refused(lib.ns_kv_extend(p, 4096, 4096, KV.MAX_ROWS + 1, None), "at most")
    refused(lib.ns_kv_fork(p, 4096, 4096, KV.MAX_ROWS + 1, None), "at most")
    refused(lib.ns_kv_free(p, None, 3, None), "NULL")
    refused(lib.ns_kv_release(p, 4096, 1, 0, 0, None), "window")
    refused(lib.ns_kv_release(p, 4096, 1, 1, -1, None), "sinks")
    refused(lib.ns_kv_compact(p, None, None, None), "page_map")
    refused(lib.ns_kv_compact(p, ctypes.byref(pool(block_tables=8192, num_cols=7, seq_lens=8192, page_refs=8192)), 4096, None),
            "differ in size")
    refused(lib.ns_kv_compact(p, ctypes.byref(pool(block_tables=8192, seq_lens=8192, page_refs=8192)), 4096, None), "share")
    refused(lib.ns_kv_copy(p, ctypes.byref(pool(block_size=8)), 4096, 4096, 1, None), "differ")
    for rc in (lib.ns_kv_extend(p, None, None, 0, None), lib.ns_kv_fork(p, None, None, 0, None),
               lib.ns_kv_free(p, None, 0, None), lib.ns_kv_release(p, None, 0, 8, 4, None),
               lib.ns_kv_copy(p, p, None, None, 0, None)):
        assert rc == 0


def test_scratch_holds_every_list():
    lib = built()
    out = ctypes.c_uint64()
    for pages in (1, 5, 100, 1024, 1025, 150000):
        assert lib.ns_kv_scratch_bytes(pages, ctypes.byref(out)) == 0
        groups = -(-pages // 1024)      # a count and 64 masks of 16 pages each
        assert out.value >= 16 + 16 * KV.MAX_ROWS + 4 * groups + 128 * groups
        assert out.value >= 4 * (4 + pages)               # a compaction's head and list
    assert lib.ns_kv_scratch_bytes(0, ctypes.byref(out)) != 0


def test_wrapper_refusals():
    built()
    k = torch.zeros(6, 16, 8, 64)
    x = torch.zeros(3, 8, 64)
    bt, one, two = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    f = torch.zeros(32)

    def refused(word, *a, **kw):
        args = list((x, x, k, k, bt, one, two, one, 16))
        for i, v in a:
            args[i] = v
        with pytest.raises(KV.KvCacheError, match=word):
            KV.store_kv_hip(*args, **kw)

    refused("must match", (1, x[:2]))
    refused("must match", (3, k[:5]))
    refused("rows", (0, x[:, :4]), (1, x[:, :4]))
    refused("block_size", (8, 8))
    refused("needs query", out=x)
    refused("inv_freq", query=x)
    refused("does not match", query=x[:2], inv_freq=f)
    refused("inv_freq", inv_freq=f[:31])
    refused("inv_freq", inv_freq=f.double())
    refused("out must match", query=x, inv_freq=f, out=x[:2])
    refused("dtype", (0, x.half()))
    refused("dtype", query=x.half(), inv_freq=f)
    refused("unit head_dim", (0, torch.zeros(3, 8, 128)[..., ::2]))
    refused("status", status=torch.zeros(1))
    refused("num_seqs", (5, two))
    refused("two dimensions", (4, one))
    refused("device tensors")
    refused("unsupported dtype", (0, x.double()), (1, x.double()), (2, k.double()), (3, k.double()))

    def no_pool(word, kc=None, vc=None, tables=torch.zeros(2, 3, dtype=torch.int32), lens=two,
                refs=torch.zeros(6, dtype=torch.int32)):
        with pytest.raises(KV.KvCacheError, match=word):
            KV.PagePool([k] if kc is None else kc, [k] if vc is None else vc, tables, lens, refs)

    no_pool("at least one", [], [])
    no_pool("as many", [k, k])
    no_pool("share shape", [k[:5]])
    no_pool("contiguous", [k.transpose(1, 2)], [k.transpose(1, 2)])
    no_pool("overlap", [k[:1].expand(6, 16, 8, 64)], [k])
    no_pool("overlap", [k], [torch.zeros(k.numel()).as_strided(k.shape, (8 * 8 * 64, 8 * 64, 64, 1))])
    no_pool("block_tables", tables=one)
    no_pool("block_tables", tables=torch.zeros((), dtype=torch.int32))
    no_pool("block_tables", tables=torch.zeros(2, 3))
    no_pool("block_tables", tables=torch.zeros(3, 2, dtype=torch.int32).t())
    no_pool("seq_lens", lens=one)
    no_pool("page_refs", refs=two)
    no_pool("16 bytes", [torch.zeros(6, 16, 1, 3)], [torch.zeros(6, 16, 1, 3)])
    no_pool("device tensors")


def test_oracle_pool_on_a_small_example():
    """The oracle itself, by hand: four pages, blocks of 2."""
    p = ORACLE.Pool([[-1, -1], [-1, -1], [-1, -1]], [0, 0, 0], [1, 0, 0, 0], 2, np.arange(8.0).reshape(4, 2))
    p.extend([1, 0], [3, 1])
    assert p.tables.tolist() == [[3, -1], [1, 2], [-1, -1]] and p.refs.tolist() == [1, 1, 1, 1]
    p.fork([1], [2])
    assert p.status == p.NO_PAGES and p.lens.tolist() == [1, 3, 0]
    p.free([0])
    p.fork([1], [2])
    assert p.tables.tolist() == [[-1, -1], [1, 2], [1, 3]] and p.refs.tolist() == [1, 2, 1, 1]
    assert p.pages.tolist() == [[0, 1], [2, 3], [4, 5], [4, 7]]
    p.free([1, 1])
    assert p.refs.tolist() == [1, 1, 0, 1]
    assert p.compact().tolist() == [0, 1, -1, 2] and p.tables.tolist() == [[-1, -1], [-1, -1], [1, 2]]
    p.release([2], 1, 0)
    assert p.tables.tolist()[2] == [-1, 2] and p.refs.tolist() == [1, 0, 1, 0]
