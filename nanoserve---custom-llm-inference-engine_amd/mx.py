"""The layer operators around attention and logits on MI355X: norms, the gated activation, and products whose weights
are held in 4 bits.

``rms_norm_hip`` does what the reference's ``RMSNorm`` (nanoserve/model/llama.py:31-37) and the residual's addition before
it (llama.py:75-85) do, in one launch; ``silu_mul_hip`` what stands between the MLP's two products (llama.py:53-56).
``mx_linear_hip`` is a linear projection (``F.linear`` without a bias: llama.py:53-56, 136-143, attention.py:97-135) with
a weight of 4-bit values, a quarter of the bytes that a decode step reads of a 16-bit one.  Its left side are rows in 8 or
4 bits, which the first two write in the same launch.

MX rows (``MxTensor``) follow the microscaling formats: blocks of 32 values share one power of two.  ``codes`` are
``float8_e4m3fn`` (rows, k) or ``float4_e2m1fn_x2`` (rows, k / 2; two values to a byte, the even one in the low half),
``scales`` are ``float8_e8m0fnu`` (rows, k / 32).  A row's ``cols`` values are padded with zeros to k, the next multiple
of 128.  A block's scale is the power of two under its largest magnitude over the largest one of the format
(2^(floor(log2 max) - 2), for 8 bits - 8); values are rounded to nearest even and held to the format's largest.  A block
with a NaN or an infinity becomes NaN as a whole.

    h = mx.rms_norm_hip(x, weight, eps, residual=residual, sum_out=residual, format="mxfp8")
    gate_up = mx.mx_linear_hip(h, w_gate_up)                      # w_gate_up = mx.quantize_mx_hip(weight, "mxfp4"), once
    a = mx.silu_mul_hip(gate_up[:, :n], gate_up[:, n:], format="mxfp8")
    x = mx.mx_linear_hip(a, w_down)

The computation runs in ``libns_mx.so`` (include/ns_mx.h); there is no other path: a missing library raises.  No call
reads anything on the host or keeps anything for the next one, and all can be captured into a graph.  No gradients are
recorded.
"""
from __future__ import annotations

import ctypes
import os
from typing import NamedTuple, Optional

import torch

from .paged_attention import host_module

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libns_mx.so")

ABI_VERSION = 1
NS_MX_F32 = 0
NS_MX_BF16 = 1
NS_MX_F16 = 2
NS_MX_FP4 = 4
NS_MX_FP8 = 8
ROW_ALIGN = 128           # values that a row is padded to a multiple of (NS_MX_ROW_ALIGN)

EXPORTS = ("ns_mx_abi_version", "ns_mx_last_error", "ns_mx_rms_norm", "ns_mx_silu_mul", "ns_mx_quantize", "ns_mx_linear",
           "ns_mx_dequantize")

_DTYPES = {torch.float32: NS_MX_F32, torch.bfloat16: NS_MX_BF16, torch.float16: NS_MX_F16}
_FORMATS = {None: 0, "mxfp4": NS_MX_FP4, "mxfp8": NS_MX_FP8}
_CODES = {"mxfp4": torch.float4_e2m1fn_x2, "mxfp8": torch.float8_e4m3fn}


class MxError(RuntimeError):
    """An argument that the library or this module refused."""


class MxTensor(NamedTuple):
    """MX rows; the calls also take a pair (codes, scales).  Products run over whole rows: what lies past ``cols`` are zero
    codes and scales that are no NaN, as every call here and ``mx_tensor`` leave them."""

    codes: torch.Tensor
    scales: torch.Tensor
    cols: int


class NsMxRows(ctypes.Structure):
    """ns_mx_rows of include/ns_mx.h, field for field."""

    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("stride_codes", ctypes.c_int64),
                ("stride_scales", ctypes.c_int64), ("format", ctypes.c_int32)]


class NsMxNormArgs(ctypes.Structure):
    """ns_mx_norm_args of include/ns_mx.h, field for field."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "residual", "weight", "rows", "sum", "out")] + [("out_mx", NsMxRows)]
                + [(n, ctypes.c_int64) for n in
                   ("n_x", "n", "stride_x", "stride_x_head", "stride_residual", "stride_residual_head", "stride_sum",
                    "stride_sum_head", "stride_out", "stride_out_head")]
                + [(n, ctypes.c_int32) for n in ("heads", "cols", "dtype", "weight_dtype")] + [("eps", ctypes.c_float)])


class NsMxGateArgs(ctypes.Structure):
    """ns_mx_gate_args of include/ns_mx.h, field for field."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("gate", "up", "rows", "out")] + [("out_mx", NsMxRows)]
                + [(n, ctypes.c_int64) for n in ("n_x", "n", "stride_gate", "stride_up", "stride_out")]
                + [("cols", ctypes.c_int32), ("dtype", ctypes.c_int32)])


class NsMxLinearArgs(ctypes.Structure):
    """ns_mx_linear_args of include/ns_mx.h, field for field."""

    _fields_ = [("x", NsMxRows), ("weight", NsMxRows), ("out", ctypes.c_void_p), ("stride_out", ctypes.c_int64),
                ("m", ctypes.c_int64), ("n", ctypes.c_int64), ("k", ctypes.c_int32), ("dtype", ctypes.c_int32)]


_LIB: Optional[ctypes.CDLL] = None
_HOST = None        # the host module, and by name the pairs of addresses of the library's functions and ns_mx_last_error


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load the HIP library (raises when it is not built: there is no fallback)."""
    global _LIB, _HOST
    if _LIB is not None:
        return _LIB
    if not os.path.exists(path):
        raise MxError(f"{path} is not built (run __graft_entry__.build())")
    lib = ctypes.CDLL(path)
    p = ctypes.c_void_p
    for name, args in (("ns_mx_abi_version", []), ("ns_mx_last_error", []),
                       ("ns_mx_rms_norm", [ctypes.POINTER(NsMxNormArgs), p]),
                       ("ns_mx_silu_mul", [ctypes.POINTER(NsMxGateArgs), p]),
                       ("ns_mx_quantize", [ctypes.POINTER(NsMxGateArgs), p]),
                       ("ns_mx_linear", [ctypes.POINTER(NsMxLinearArgs), p]),
                       ("ns_mx_dequantize", [ctypes.POINTER(NsMxRows), ctypes.c_int64, ctypes.c_int32, p, ctypes.c_int64,
                                             ctypes.c_int32, p])):
        f = getattr(lib, name)
        f.restype, f.argtypes = ctypes.c_int, args
    lib.ns_mx_last_error.restype = ctypes.c_char_p
    if lib.ns_mx_abi_version() != ABI_VERSION:
        raise MxError(f"ABI {lib.ns_mx_abi_version()} in {path}, expected {ABI_VERSION}")
    host = host_module(MxError)
    host.set_errors(None, None, MxError)
    at = {n: ctypes.cast(getattr(lib, n), p).value for n in EXPORTS}
    _HOST = (host, {n: (at["ns_mx_" + n], at["ns_mx_last_error"])
                    for n in ("rms_norm", "silu_mul", "quantize", "dequantize", "linear")})
    _LIB = lib
    return lib


def _on(t, stream):
    """(HIP stream handle, context or None) of a call on a tensor's device: its current stream, a torch stream or a raw
    handle (0: the default stream).  Inside the context the call's results are made on that stream."""
    dev = t.get_device() if isinstance(t, torch.Tensor) else -1
    if dev < 0:
        return 0, None        # refused by the call
    if stream is None:
        if dev == torch._C._cuda_getDevice():    # a CUDA tensor is there, so torch has made the device ready
            return torch._C._cuda_getCurrentRawStream(dev), None
        s = torch.cuda.current_stream(dev)
    elif isinstance(stream, torch.cuda.Stream):
        if stream.device_index != dev:
            raise MxError(f"the stream is one of device {stream.device_index}, the tensors are on device {dev}")
        s = stream
    elif int(stream) == 0:
        s = torch.cuda.default_stream(dev)
    else:
        s = torch.cuda.ExternalStream(int(stream), device=dev)
    return s.cuda_stream, torch.cuda.stream(s)


def _run(call, t, stream, *args):
    handle, context = _on(t, stream)
    if context is None:
        return call(*args, handle)
    with context:
        return call(*args, handle)


def _format(format):
    if format not in _FORMATS:
        raise MxError(f"format must be None, \"mxfp4\" or \"mxfp8\", not {format!r}")
    return _FORMATS[format]


def _dtype(dtype):
    if dtype not in _DTYPES:
        raise MxError(f"unsupported dtype {dtype} (float32, bfloat16, float16)")
    return _DTYPES[dtype]


def _pair(t, name):
    """(codes, scales, cols or None) of an MxTensor or a pair."""
    if not isinstance(t, (tuple, list)) or not 2 <= len(t) <= 3:
        raise MxError(f"{name} must be an MxTensor or a pair (codes, scales)")
    return t if len(t) == 3 else (*t, None)


def _out(out, format):
    """The codes and scales, or the tensor, that a result goes to."""
    if out is None:
        return None, None
    return _pair(out, "out")[:2] if format is not None else (out, None)


def rms_norm_hip(x, weight, eps: float, *, residual=None, sum_out=None, rows=None, format: Optional[str] = None, out=None,
                 stream=None):
    """h * weight / sqrt(mean(h^2) + eps) over the last dimension, h = x or x + residual (rounded to their type).

    x (n, cols) or (n, heads, cols), each head a norm of its own, float32, bfloat16 or float16 with a unit stride along
    cols; ``residual`` like x; ``weight`` (cols) of x's type or float32.  ``sum_out``, like the result in x's type,
    receives h (the next residual).  ``rows``, a contiguous int64 tensor: only these rows are taken, in its order (a
    step's sample positions); an index outside x gives a row of NaN.  With ``format`` the result is an ``MxTensor``
    (two-dimensional x), else a tensor like x.  It is computed in float32, the squares' sum in float64, and rounded once.
    ``out`` takes the result; ``out`` and ``sum_out`` may be x or residual themselves where no rows are picked, and lie
    apart from everything read otherwise.  ``stream``: a ``torch.cuda.Stream`` or a raw HIP stream handle, default the
    current stream.
    """
    if _LIB is None:
        load()
    host, calls = _HOST
    fmt = _format(format)
    to, scales = _out(out, format)
    got = _run(host.rms_norm, x, stream, *calls["rms_norm"], x, weight, eps, residual, sum_out, rows, fmt, to, scales)
    return got if fmt == 0 else MxTensor(*got, x.shape[1])


def silu_mul_hip(gate, up, *, format: Optional[str] = None, out=None, stream=None):
    """silu(gate) * up = gate / (1 + exp(-gate)) * up in float32, rounded once to the inputs' type or, with ``format``, to
    MX rows.  gate and up (n, cols), as the two halves of a fused projection's rows are; ``out`` may be one of them."""
    if _LIB is None:
        load()
    host, calls = _HOST
    if up is None:
        raise MxError("up must be a tensor")
    fmt = _format(format)
    to, scales = _out(out, format)
    got = _run(host.gate, gate, stream, *calls["silu_mul"], gate, up, None, fmt, to, scales)
    return got if fmt == 0 else MxTensor(*got, gate.shape[1])


def quantize_mx_hip(x, format: str = "mxfp4", *, rows=None, out=None, stream=None) -> MxTensor:
    """x (n, cols) as MX rows; ``rows`` as for ``rms_norm_hip``.  A weight (out features, in features) is quantized once, in
    "mxfp4", for ``mx_linear_hip``."""
    if _LIB is None:
        load()
    host, calls = _HOST
    if format is None:
        raise MxError("format must be \"mxfp4\" or \"mxfp8\"")
    fmt = _format(format)
    to, scales = _out(out, format)
    got = _run(host.gate, x, stream, *calls["quantize"], x, None, rows, fmt, to, scales)
    return MxTensor(*got, x.shape[1])


def dequantize_mx_hip(t, dtype=torch.bfloat16, *, out=None, stream=None):
    """The values that MX rows stand for, (n, cols) of ``dtype`` (rounded to nearest even where it does not hold them)."""
    if _LIB is None:
        load()
    host, calls = _HOST
    codes, scales, cols = _pair(t, "t")
    return _run(host.dequantize, codes, stream, *calls["dequantize"], codes, scales, -1 if cols is None else cols, _dtype(dtype),
                out)


def mx_linear_hip(x, weight, *, dtype=torch.bfloat16, out=None, stream=None):
    """x @ weight.T, (m, n) of ``dtype``: x MX rows in either format, (m, cols), and weight MX rows in 4 bits, (n, cols).
    The products of the values that the codes stand for are exact, their sums are float32, rounded once to ``dtype``."""
    if _LIB is None:
        load()
    host, calls = _HOST
    xc, xs, x_cols = _pair(x, "x")
    wc, ws, w_cols = _pair(weight, "weight")
    if x_cols is not None and w_cols is not None and x_cols != w_cols:
        raise MxError(f"x's rows of {x_cols} values do not match the weight's of {w_cols}")
    return _run(host.linear, xc, stream, *calls["linear"], xc, xs, wc, ws, _dtype(dtype), out)


def mx_tensor(codes, scales, cols: Optional[int] = None) -> MxTensor:
    """MX rows as other programs store them, laid out for these calls (a copy where they are not so already): codes
    (rows, k), ``float8_e4m3fn``, or (rows, k / 2), ``float4_e2m1fn_x2`` or uint8 of the same bits, scales (rows, k / 32),
    ``float8_e8m0fnu`` or uint8, for any k that is a multiple of 32; ``cols`` (default k): the values in use.  What is stored
    past them is left out: with ``cols`` below k device tensors are copied (nothing is read on the host to see whether there
    is anything), host tensors where it would enter a product."""
    if not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor):
        raise MxError("codes and scales must be tensors")
    if codes.dtype is torch.uint8:
        codes = codes.view(torch.float4_e2m1fn_x2)
    if scales.dtype is torch.uint8:
        scales = scales.view(torch.float8_e8m0fnu)
    if codes.dtype not in _CODES.values() or scales.dtype is not torch.float8_e8m0fnu:
        raise MxError(f"codes of {codes.dtype} and scales of {scales.dtype} are no MX rows")
    per = 2 if codes.dtype is torch.float4_e2m1fn_x2 else 1
    if codes.dim() != 2 or scales.dim() != 2:
        raise MxError("codes and scales must have two dimensions")
    n, k = codes.shape[0], codes.shape[1] * per
    if k == 0 or k % 32 != 0 or tuple(scales.shape) != (n, k // 32) or scales.device != codes.device:
        raise MxError(f"codes {tuple(codes.shape)} need scales {(n, k // 32)} on their device, got {tuple(scales.shape)}")
    cols = k if cols is None else int(cols)
    if not 0 < cols <= k:
        raise MxError(f"cols must lie in 1 .. {k}, not {cols}")

    def laid_out(t, width, unit, used, last, harmful):
        """Rows of ``width`` bytes, those from ``used`` on zero and of the one before only the bits of ``last``."""
        b = t.view(torch.uint8)
        fits = t.shape[1] == width and t.stride(1) == 1 and (n < 2 or t.stride(0) % unit == 0) and t.data_ptr() % unit == 0
        if fits and (cols == k or not (t.is_cuda or harmful(b[:, used:]).any() or (b[:, used - 1] & (255 - last)).any())):
            return t
        new = torch.zeros((n, width), dtype=torch.uint8, device=t.device)
        new[:, :used] = b[:, :used]
        if last != 255:
            new[:, used - 1] &= last
        return new.view(t.dtype)

    wide = -(-k // ROW_ALIGN) * ROW_ALIGN
    half = per == 2 and cols % 2 == 1        # the last value in use shares its byte with one that is not
    return MxTensor(laid_out(codes, wide // per, 16, -(-cols // per), 15 if half else 255, lambda past: past != 0),
                    laid_out(scales, wide // 32, 4, -(-cols // 32), 255, lambda past: past == 255), cols)
