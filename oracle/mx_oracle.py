"""CPU oracle of the layer operators: norms, the gated activation, MX rows and their products.

TEST INFRASTRUCTURE ONLY: imported by ``tests/`` as the oracle of the HIP kernels, never by the product.

Everything is float64; MX codes are handled as the values that they stand for, looked up in tables written out from the
formats' definitions.  ``rms_norm`` follows nanoserve/model/llama.py:31-37, ``silu_mul`` llama.py:53-56.
"""
from __future__ import annotations

import numpy as np

BLOCK, ALIGN = 32, 128
EMAX = {"mxfp4": 2, "mxfp8": 8}
MOST = {"mxfp4": 6.0, "mxfp8": 448.0}


def _e2m1():
    pos = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return np.array(pos + [-x for x in pos])


def _e4m3():
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = np.nan if (c & 127) == 127 else x
        if c >= 128:
            v[c] = -v[c]
    return v


E2M1, E4M3 = _e2m1(), _e4m3()


def padded(x):
    """x with zeros up to a multiple of 128 columns."""
    x = np.asarray(x, dtype=np.float64)
    return np.concatenate([x, np.zeros((x.shape[0], -x.shape[1] % ALIGN))], axis=1)


def block_scales(x, fmt):
    """The exponents of the blocks of x (padded); None stands for NaN and is returned as 128."""
    blocks = np.abs(padded(x)).reshape(x.shape[0], -1, BLOCK)
    fine = np.isfinite(blocks).all(-1)
    most = np.where(fine, blocks.max(-1, initial=0.0, where=np.isfinite(blocks)), 1.0)
    _, e = np.frexp(most)
    e = np.where(most > 0, np.maximum(e - 1 - EMAX[fmt], -127), -127)
    return np.where(fine, e, 128)


def at_scales(x, e, fmt):
    """The values of x (padded) rounded to the format under the blocks' exponents e, as what they stand for (NaN for 128)."""
    grid = np.sort(E2M1[:8] if fmt == "mxfp4" else E4M3[:127])
    x = padded(x).reshape(x.shape[0], -1, BLOCK)
    with np.errstate(invalid="ignore", over="ignore"):
        v = x / np.ldexp(1.0, e)[..., None]
    a = np.minimum(np.where(np.isfinite(v), np.abs(v), 0.0), MOST[fmt])
    up = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    lo, hi = grid[up - 1], grid[up]
    mid = (lo + hi) / 2
    # the grid's entries are the codes in order: of two at the same distance the even code
    got = np.where((a > mid) | ((a == mid) & (up % 2 == 0)), hi, lo)
    got = np.where(v < 0, -got, got) * np.ldexp(1.0, e)[..., None]
    return np.where((e == 128)[..., None], np.nan, got).reshape(x.shape[0], -1)


def quantize(x, fmt):
    """(values, exponents) of MX rows of x."""
    e = block_scales(x, fmt)
    return at_scales(x, e, fmt), e


def values(codes, scales, fmt):
    """The values of code bytes and scale bytes as stored."""
    codes = np.asarray(codes, dtype=np.int64)
    if fmt == "mxfp4":
        v = E2M1[np.stack([codes & 15, codes >> 4], axis=-1).reshape(codes.shape[0], -1)]
    else:
        v = E4M3[codes]
    s = np.asarray(scales, dtype=np.int64)
    e = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return (v.reshape(v.shape[0], -1, BLOCK) * e[..., None]).reshape(v.shape[0], -1)


def rms_norm(h, weight, eps):
    """h (float64, as the sum was rounded) of any leading shape."""
    with np.errstate(invalid="ignore", divide="ignore"):
        return h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * weight


def silu_mul(gate, up):
    with np.errstate(over="ignore", invalid="ignore"):
        return np.where(gate < 0, gate * np.exp(np.minimum(gate, 0)) / (1 + np.exp(np.minimum(gate, 0))),
                        gate / (1 + np.exp(-np.maximum(gate, 0)))) * up


def linear(x, w):
    """(x @ w.T, |x| @ |w|.T) of values."""
    return x @ w.T, np.abs(x) @ np.abs(w).T
