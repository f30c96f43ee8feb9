"""CPU checks of the layer operators' library: exports, struct layouts, refusals before any launch, and the oracle."""
import ctypes
import os
import re
import subprocess
import tempfile

import numpy as np
import pytest
import torch

from conftest import ROOT, pkg
from mx_cases import codes_of, small_integers
from oracle import mx_oracle as ORACLE

MX = pkg("mx")
HEADER = os.path.join(ROOT, "include", "ns_mx.h")


def built():
    if not os.path.exists(MX.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    return MX.load()


def test_exports_and_version():
    txt = open(HEADER).read()
    names = sorted(set(re.findall(r"^\s*(?:int|const char\*)\s+(ns_\w+)\s*\(", txt, flags=re.M)))
    assert names == sorted(MX.EXPORTS)
    lib = built()
    for name in names:
        assert hasattr(lib, name), name
    define = lambda n: int(re.search(rf"#define {n} (\d+)", txt).group(1))  # noqa: E731
    assert lib.ns_mx_abi_version() == MX.ABI_VERSION == define("NS_MX_ABI_VERSION")
    assert MX.ROW_ALIGN == define("NS_MX_ROW_ALIGN") == ORACLE.ALIGN
    for name in ("F32", "BF16", "F16", "FP4", "FP8"):
        assert getattr(MX, "NS_MX_" + name) == define("NS_MX_" + name)


@pytest.mark.parametrize("struct,cls", [("ns_mx_rows", MX.NsMxRows), ("ns_mx_norm_args", MX.NsMxNormArgs),
                                        ("ns_mx_gate_args", MX.NsMxGateArgs), ("ns_mx_linear_args", MX.NsMxLinearArgs)])
def test_struct_layout_matches_header(struct, cls):
    txt = open(HEADER).read()
    body = txt[txt.index(f"typedef struct {struct} {{"):txt.index(f"}} {struct};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for decl in re.findall(r"^\s*([^/{}]+?);", body, flags=re.M):
        names += [n.strip().lstrip("*") for n in re.sub(r"^.*?\b(\w+)\s*(,|$)", r"\1\2", decl, count=1).split(",")]
    assert names == [f[0] for f in cls._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"ns_mx.h\"\nint main(void) {\n"
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


def rows(**kw):
    r = MX.NsMxRows(4096, 4096, 256, 8, MX.NS_MX_FP8)
    for n, v in kw.items():
        setattr(r, n, v)
    return r


def norm_args(**kw):
    a = MX.NsMxNormArgs(x=4096, weight=4096, out=4096, n_x=4, n=4, stride_x=200, stride_out=200, heads=1, cols=200,
                        dtype=MX.NS_MX_BF16, weight_dtype=MX.NS_MX_BF16, eps=1e-5)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def gate_args(**kw):
    a = MX.NsMxGateArgs(gate=4096, up=4096, out=4096, n_x=4, n=4, stride_gate=200, stride_up=200, stride_out=200, cols=200,
                        dtype=MX.NS_MX_BF16)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def linear_args(**kw):
    a = MX.NsMxLinearArgs(x=rows(), weight=rows(format=MX.NS_MX_FP4, stride_codes=128), out=4096, stride_out=16, m=4, n=16,
                          k=256, dtype=MX.NS_MX_BF16)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def refused(name, args, word):
    lib = built()
    assert getattr(lib, name)(ctypes.byref(args), None) != 0
    assert word in lib.ns_mx_last_error().decode(), lib.ns_mx_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=7), "dtype"), (dict(weight_dtype=MX.NS_MX_F16), "weight_dtype"), (dict(n=-1), "n and n_x"),
    (dict(heads=0), "heads"), (dict(cols=0), "cols"), (dict(cols=(1 << 30) + 1), "cols"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(x=None), "NULL"), (dict(weight=None), "NULL"), (dict(n=3), "as many"),
    (dict(rows=4096, n_x=0), "empty"), (dict(out=None), "out"), (dict(out_mx=rows()), "one of"),
    (dict(out=None, out_mx=rows(), heads=2), "heads"), (dict(out=None, out_mx=rows(format=3)), "format"),
    (dict(out=None, out_mx=rows(codes=None)), "NULL"), (dict(out=None, out_mx=rows(codes=4104)), "16-byte"),
    (dict(out=None, out_mx=rows(stride_codes=264)), "16-byte"), (dict(out=None, out_mx=rows(stride_codes=192)), "wide"),
    (dict(out=None, out_mx=rows(stride_scales=6)), "4-byte"), (dict(out=None, out_mx=rows(stride_scales=4)), "wide"),
    (dict(out=None, out_mx=rows(scales=4098)), "4-byte"), (dict(stride_x=-1), "negative"),
    (dict(stride_sum_head=-1), "negative")])
def test_norm_refusals(kw, word):
    refused("ns_mx_rms_norm", norm_args(**kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=4), "dtype"), (dict(n=-1), "n and n_x"), (dict(cols=0), "cols"), (dict(cols=(1 << 26) + 1), "cols"),
    (dict(gate=None), "NULL"), (dict(up=None), "NULL"), (dict(rows=4096), "rows"), (dict(n=5), "as many"),
    (dict(out=None), "out"), (dict(out_mx=rows()), "one of"), (dict(stride_up=-2), "negative")])
def test_gate_refusals(kw, word):
    refused("ns_mx_silu_mul", gate_args(**kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(up=4096), "neither"), (dict(out=4096, out_mx=rows(format=0)), "neither"), (dict(out_mx=rows(format=0)), "out"),
    (dict(out_mx=rows(format=5)), "format"), (dict(n=5), "as many"), (dict(rows=4096, n_x=0), "empty")])
def test_quantize_refusals(kw, word):
    refused("ns_mx_quantize", gate_args(**{**dict(up=None, out=None, out_mx=rows()), **kw}), word)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=8), "dtype"), (dict(m=-1), "m and n"), (dict(n=1 << 31), "m and n"), (dict(k=0), "k must"),
    (dict(k=192), "k must"), (dict(x=rows(format=0)), "format"), (dict(x=rows(codes=4100)), "16-byte"),
    (dict(x=rows(stride_codes=128)), "wide"), (dict(x=rows(stride_scales=4)), "wide"),
    (dict(weight=rows()), "NS_MX_FP4"), (dict(weight=rows(format=MX.NS_MX_FP4, scales=None)), "NULL"),
    (dict(weight=rows(format=MX.NS_MX_FP4, stride_codes=112)), "wide"), (dict(out=None), "out"),
    (dict(stride_out=15), "stride_out"), (dict(x=rows(stride_codes=1 << 23)), "2^23"),
    (dict(weight=rows(format=MX.NS_MX_FP4, stride_scales=1 << 23)), "2^23")])
def test_linear_refusals(kw, word):
    refused("ns_mx_linear", linear_args(**kw), word)


def test_dequantize_refusals_and_empty_calls():
    lib = built()

    def off(word, r=None, n=4, cols=200, out=4096, stride=200, dtype=MX.NS_MX_BF16):
        assert lib.ns_mx_dequantize(ctypes.byref(r or rows()), n, cols, out, stride, dtype, None) != 0
        assert word in lib.ns_mx_last_error().decode()

    off("dtype", dtype=8)
    off("n must", n=-1)
    off("cols", cols=0)
    off("out", out=None)
    off("stride_out", stride=-1)
    off("stride_out", stride=199)
    off("format", rows(format=1))
    off("wide", rows(stride_codes=128))
    assert lib.ns_mx_dequantize(None, 1, 1, 4096, 1, 0, None) != 0
    assert lib.ns_mx_dequantize(ctypes.byref(rows()), 0, 200, None, 200, 0, None) == 0
    for name, args in (("ns_mx_rms_norm", norm_args(n=0, n_x=0, x=None, out=None)), ("ns_mx_silu_mul", gate_args(n=0, n_x=0)),
                       ("ns_mx_quantize", gate_args(n=0, n_x=0, up=None, out=None)), ("ns_mx_linear", linear_args(m=0)),
                       ("ns_mx_linear", linear_args(n=0))):
        assert getattr(lib, name)(ctypes.byref(args), None) == 0
        assert getattr(lib, name)(None, None) != 0


def test_wrapper_refusals():
    built()
    x, w, idx = torch.zeros(4, 256), torch.zeros(256), torch.zeros(3, dtype=torch.int64)
    half = torch.zeros(4, 512)
    q8, q4 = (small_integers(1, 4, 256, f)[0] for f in ("mxfp8", "mxfp4"))

    def no(f, word, *a, **kw):
        with pytest.raises(MX.MxError, match=word):
            f(*a, **kw)

    norm = MX.rms_norm_hip
    no(norm, "tensor", None, w, 1e-5)
    no(norm, "dimensions", x[0], w, 1e-5)
    no(norm, "dtype", x.double(), w, 1e-5)
    no(norm, "columns", x[:, :0], w[:0], 1e-5)
    no(norm, "unit stride", half[:, ::2], w, 1e-5)
    no(norm, "weight", x, w[:255], 1e-5)
    no(norm, "weight", x, w.half(), 1e-5)
    no(norm, "weight", x, torch.zeros(512)[::2], 1e-5)
    no(norm, "eps", x, w, -1e-5)
    no(norm, "eps", x, w, float("nan"))
    no(norm, "residual", x, w, 1e-5, residual=x[:3])
    no(norm, "residual", x, w, 1e-5, residual=x.half())
    no(norm, "residual", x, w, 1e-5, residual=half[:, ::2])
    no(norm, "sum_out", x, w, 1e-5, sum_out=x[:3])
    no(norm, "sum_out", x, w, 1e-5, rows=idx, sum_out=x)
    no(norm, "rows", x, w, 1e-5, rows=idx.int())
    no(norm, "rows", x, w, 1e-5, rows=idx[None])
    no(norm, "rows", x, w, 1e-5, rows=torch.zeros(6, dtype=torch.int64)[::2])
    no(norm, "rows", x[:0], w, 1e-5, rows=idx)
    no(norm, "rows", x[:, None], w, 1e-5, rows=idx)
    no(norm, "format", x, w, 1e-5, format="mxfp6")
    no(norm, "format", x[:, None], w, 1e-5, format="mxfp8")
    no(norm, "out", x, w, 1e-5, out=x[:3])
    no(norm, "out", x, w, 1e-5, out=x.half())
    no(norm, "out", x, w, 1e-5, out=half[:, ::2])
    no(norm, "MxTensor", x, w, 1e-5, out=x, format="mxfp8")
    no(norm, "format", x, w, 1e-5, out=q4, format="mxfp8")
    no(norm, "shape", x[:3], w, 1e-5, out=q8, format="mxfp8")
    no(norm, "device tensors", x, w, 1e-5)
    gated = MX.silu_mul_hip
    no(gated, "tensor", x, None)
    no(gated, "up", x, x[:3])
    no(gated, "up", x, x.half())
    no(gated, "dimensions", x[0], x[0])
    no(gated, "unit stride", half[:, ::2], half[:, 1::2])
    no(gated, "format", x, x, format="fp8")
    no(gated, "device tensors", x, x)
    quant = MX.quantize_mx_hip
    no(quant, "format", x, None)
    no(quant, "dimensions", x[None])
    no(quant, "rows", x, rows=idx.int())
    no(quant, "out", x, "mxfp8", out=q4)
    no(quant, "device tensors", x)
    values = MX.dequantize_mx_hip
    no(values, "MxTensor", x)
    no(values, "dtype", q8, torch.float64)
    no(values, "cols", (*q8[:2], 257))
    no(values, "codes", (x, q8.scales))
    no(values, "scales", (q8.codes, q8.scales.view(torch.uint8)))
    no(values, "padded", (q8.codes[:, :192], q8.scales[:, :6]))
    no(values, "padded", (q8.codes, q8.scales[:, :4]))
    no(values, "as many", (q8.codes[:3], q8.scales))
    no(values, "out", q8, out=x)
    no(values, "device tensors", q8)
    linear = MX.mx_linear_hip
    no(linear, "x must", x, q4)
    no(linear, "weight must", q8, w)
    no(linear, "weight", q8, q8)
    no(linear, "match", q8, small_integers(2, 4, 384, "mxfp4")[0])
    no(linear, "match", small_integers(2, 4, 200, "mxfp8")[0], q4)
    no(linear, "dtype", q8, q4, dtype=torch.int32)
    no(linear, "out", q8, q4, out=torch.zeros(4, 4))
    no(linear, "unit stride", q8, q4, dtype=torch.float32, out=torch.zeros(4, 8)[:, ::2])
    no(linear, "device tensors", q8, q4)


def test_mx_tensor_lays_rows_out():
    full, v = small_integers(3, 5, 160, "mxfp4")
    narrow = MX.MxTensor(full.codes.view(torch.uint8)[:, :80].contiguous(), full.scales.view(torch.uint8)[:, :5].contiguous(), 160)
    got = MX.mx_tensor(narrow.codes, narrow.scales)
    assert got.cols == 160 and got.codes.shape == (5, 128) and got.scales.shape == (5, 8)
    assert np.array_equal(codes_of(got)[0], v)
    same = MX.mx_tensor(full.codes, full.scales, 160)
    assert same.codes is full.codes and same.scales is full.scales and same.cols == 160
    q8, v8 = small_integers(4, 3, 128, "mxfp8")
    shifted = torch.zeros(3 * 128 + 8, dtype=torch.uint8)[8:].view(3, 128)      # not at 16 bytes
    shifted.copy_(q8.codes.view(torch.uint8))
    got = MX.mx_tensor(shifted.view(torch.float8_e4m3fn), q8.scales)
    assert got.codes.data_ptr() % 16 == 0 and np.array_equal(codes_of(got)[0], v8)
    for bad in ((q8.codes[:, :100], q8.scales), (q8.codes, q8.scales[:2]), (q8.codes[0], q8.scales[0]),
                (q8.codes.float(), q8.scales), (q8.codes, q8.scales.float()), (None, q8.scales)):
        with pytest.raises(MX.MxError):
            MX.mx_tensor(*bad)
    with pytest.raises(MX.MxError, match="cols"):
        MX.mx_tensor(q8.codes, q8.scales, 129)


def test_oracle_values_and_rounding():
    """The oracle itself: torch's own 8-bit type, ties by hand, and the scale at the powers of two."""
    every = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(ORACLE.E4M3, every.view(torch.float8_e4m3fn).double().numpy(), equal_nan=True)
    x = np.zeros((1, 128))
    x[0, :8] = [6, 5, 0.25, 0.75, -2.5, 3.5, 7.9, -0.25]
    v, e = ORACLE.quantize(x, "mxfp4")
    assert e[0, 0] == 0 and v[0, :8].tolist() == [6, 4, 0, 1, -2, 4, 6, 0]
    for most, want in ((1.0, -2), (1.999, -2), (2.0, -1), (2.0 ** -140, -127), (0.0, -127), (np.inf, 128), (np.nan, 128)):
        x[0, :8] = 0
        x[0, 3] = -most
        assert ORACLE.block_scales(x, "mxfp4")[0, 0] == want
    y = np.random.default_rng(0).standard_normal((20, 256)) * 300
    y[:, 0] = 447.9
    v, e = ORACLE.quantize(np.clip(y, -448, 448), "mxfp8")
    want = torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn).double().numpy()
    assert (e[:, 0] == 0).all() and np.array_equal(v[:, :32], want[:, :32])
