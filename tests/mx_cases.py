"""Inputs and bounds of the layer operators' tests.

Bounds, with u = 2^-24 (float32 rounds a result by at most u of it):
* norm: the sum is float64 over values (float32) or over pairs whose sum is rounded once (16 bits: u of the sum, half of it of
  the root), the root is float64, the factor is rounded once (u), two products follow (2 u): 3.5 u of the value, and 4 u
  leaves the float64 parts their room.
* gated: exp within 3 u (2^t by the instruction within 1 ulp, 2 u, and the product with what t's rounding left), 1 + e adds
  its own u (exp's error enters the quotient e / (1 + e) less than once over), the reciprocal and its product with e u each,
  and the two products after it: 3 + 1 + 1 + 1 + 1 + 1 = 8 u.  Where the exponential or a product
  falls below the normal numbers, 2^-149 of it is lost, times |gate up|.
* a rounding to the type: half a unit in its last place (float32's is the last product's, counted above).
* a result in MX rows: the value before rounding is within those bounds, so the block's exponent is one of the two ends',
  and under it each code lies between the codes of the two ends.
* products: values exact, so k terms in float32 in any order lose at most (k - 1) u of the sum of their magnitudes where
  each addition rounds, twice that where it cuts; 2 k u is taken.  A 16-bit result of 8-bit rows may lose each product's part
  below 2^-13 of the largest of its eight neighbours besides: at most 7 2^-13 of that one, which has a test of its own."""
import numpy as np
import torch

from conftest import pkg
from oracle import mx_oracle as ORACLE

U = 2.0 ** -24
BITS = {torch.bfloat16: 8, torch.float16: 11, torch.float32: 24}
LEAST = {torch.bfloat16: -133, torch.float16: -24, torch.float32: -149}   # exponent of the smallest subnormal
NORM, GATED = 4 * U, 8 * U
FORMATS = ("mxfp4", "mxfp8")
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def f64(t):
    return t.detach().double().cpu().numpy()


def bits(t):
    return t.view(torch.uint8).cpu().numpy()


def codes_of(q):
    """(values, exponents) of an MxTensor on any device, from its bytes."""
    fmt = "mxfp8" if q.codes.dtype is torch.float8_e4m3fn else "mxfp4"
    return ORACLE.values(bits(q.codes), bits(q.scales), fmt), bits(q.scales).astype(np.int64) - 127


def half_ulp(x, dtype):
    _, e = np.frexp(np.abs(x))
    return np.ldexp(0.5, np.maximum(e - BITS[dtype], LEAST[dtype]))


def assert_near(got, want, dtype, rel, floor=0.0):
    """A result in a type: NaN and infinities where the formula has them, else within the bound."""
    got = f64(got)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    most = float(torch.finfo(dtype).max)
    fine = np.isfinite(want) & (np.abs(want) <= most)
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    g, w = got[fine], want[fine]
    last = 0.0 if dtype is torch.float32 else half_ulp(np.maximum(np.abs(w), np.abs(np.where(np.isinf(g), w, g))), dtype)
    bound = last + rel * np.abs(w) + np.broadcast_to(floor, want.shape)[fine] + 2.0 ** -149
    bad = np.abs(g - w) > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} off, the worst by {np.abs(g - w).max()}"


def assert_mx(q, want, fmt, rel, floor=0.0):
    """A result in MX rows of the values `want` (before rounding)."""
    got, e = codes_of(q)
    n, cols = want.shape
    wide = -(-cols // 128) * 128
    assert got.shape == (n, wide) and q.cols == cols and e.shape == (n, wide // 32)
    off = rel * np.abs(want) + floor
    grown, shrunk = np.abs(want) + off, np.maximum(np.abs(want) - off, 0)
    e_hi, e_lo = ORACLE.block_scales(grown, fmt), ORACLE.block_scales(shrunk, fmt)
    assert ((e == e_hi) | (e == e_lo)).all()
    a, b = ORACLE.at_scales(want - off, e, fmt), ORACLE.at_scales(want + off, e, fmt)
    nan = np.repeat(e == 128, 32, axis=1)
    assert np.array_equal(np.isnan(got), nan)
    assert ((got >= np.minimum(a, b)) & (got <= np.maximum(a, b)) | nan).all()
    assert not got[:, cols:][~nan[:, cols:]].any()
    if wide - cols >= 32:       # whole blocks of padding
        pad = slice(-(-cols // 32), None)
        assert (e[:, pad] == -127).all()
    if nan.any():               # the codes of a NaN block are zero
        raw = bits(q.codes)
        raw = raw if fmt == "mxfp8" else np.stack([raw & 15, raw >> 4], -1).reshape(n, -1)
        assert not raw[nan].any()


def hidden(seed, rows, cols, dtype=torch.bfloat16, size=1.0):
    """Rows of different sizes with a few large channels, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * size
    x *= torch.randn(cols, generator=g).mul(0.7).exp() * torch.randn(rows, 1, generator=g).mul(0.5).exp()
    return x.to(dtype)


def small_integers(seed, rows, cols, fmt, device=None):
    """MX rows whose values are small whole multiples of a power of two, so that their products sum exactly in float32:
    (MxTensor on the CPU or device, values).  Codes of all magnitudes up to 6 or 8, scales of 2^-2 .. 2^2."""
    MX = pkg("mx")
    r = np.random.default_rng(seed)
    wide = -(-cols // 128) * 128
    if fmt == "mxfp4":
        codes = r.integers(0, 16, (rows, wide))
    else:
        grid = np.array([c for c in range(256) if abs(ORACLE.E4M3[c]) in (0, 0.5, 1, 1.5, 2, 3, 4, 5, 6, 7, 8)])
        codes = grid[r.integers(0, len(grid), (rows, wide))]
    codes[:, cols:] = 0
    scales = r.integers(125, 130, (rows, wide // 32))
    if fmt == "mxfp4":
        codes = codes[:, ::2] | codes[:, 1::2] << 4
    v = ORACLE.values(codes, scales, fmt)
    c = torch.from_numpy(codes.astype(np.uint8)).view(torch.float8_e4m3fn if fmt == "mxfp8" else torch.float4_e2m1fn_x2)
    s = torch.from_numpy(scales.astype(np.uint8)).view(torch.float8_e8m0fnu)
    if device is not None:
        c, s = c.to(device), s.to(device)
    return MX.MxTensor(c, s, cols), v
