"""``mx_tensor``: rows as other programs store them, whose bytes past the values in use may be anything."""
import numpy as np
import pytest
import torch

from conftest import pkg
from mx_cases import FORMATS, codes_of
from oracle import mx_oracle as ORACLE

MX = pkg("mx")


def stored(seed, rows, k, fmt):
    """(codes, scales) of k values a row, every byte pattern but NaN's among them, and their values."""
    r = np.random.default_rng(seed)
    codes = r.integers(0, 256, (rows, k if fmt == "mxfp8" else k // 2))
    if fmt == "mxfp8":
        codes[codes % 128 == 127] = 126
    scales = r.integers(100, 150, (rows, k // 32))
    return codes, scales, ORACLE.values(codes, scales, fmt)


def as_rows(codes, scales, fmt, device="cpu"):
    c = torch.from_numpy(codes.astype(np.uint8)).to(device)
    s = torch.from_numpy(scales.astype(np.uint8)).to(device).view(torch.float8_e8m0fnu)
    return (c.view(torch.float8_e4m3fn) if fmt == "mxfp8" else c), s


def check(device):
    for fmt in FORMATS:
        for k, cols in ((128, 100), (256, 128), (256, 129), (256, 1), (160, 131), (416, 383), (128, 127), (64, 33), (128, 96)):
            codes, scales, v = stored(k + cols, 5, k, fmt)
            scales[2, -(-cols // 32):] = 255                      # blocks past the values in use
            if fmt == "mxfp8":
                codes[3, cols:] = 127
            given = as_rows(codes, scales, fmt, device)
            before = [t.view(torch.uint8).clone() for t in given]
            q = MX.mx_tensor(*given, cols)
            assert q.cols == cols and q.codes.device == given[0].device
            got, e = codes_of(q)
            assert np.array_equal(got[:, :cols], v[:, :cols]) and not got[:, cols:].any(), (fmt, k, cols)
            assert (e[:, -(-cols // 32):] != 128).all()
            assert all(torch.equal(t.view(torch.uint8), b) for t, b in zip(given, before))   # the caller's stay as they were


def test_what_lies_past_the_values_in_use_is_cleared():
    check("cpu")


@pytest.mark.gpu
def test_what_lies_past_the_values_in_use_is_cleared_on_the_device(device):
    check(device)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_a_product_is_that_of_the_values_in_use(device, fmt):
    """Both sides' rows end in bytes that mean nothing: the product is the one of what ``dequantize_mx_hip`` gives."""
    for m, n, k, cols in ((1, 40, 128, 100), (20, 70, 256, 131), (200, 33, 160, 129)):
        (xc, xs, _), (wc, ws, _) = stored(m, m, k, fmt), stored(n, n, k, "mxfp4")
        xs[:, -(-cols // 32):], ws[::2, -(-cols // 32):] = 255, 255
        x, w = MX.mx_tensor(*as_rows(xc, xs, fmt, device), cols), MX.mx_tensor(*as_rows(wc, ws, "mxfp4", device), cols)
        xv, wv = (MX.dequantize_mx_hip(t, torch.float32).cpu().double().numpy() for t in (x, w))
        want, total = ORACLE.linear(xv, wv)
        got = MX.mx_linear_hip(x, w, dtype=torch.float32).cpu().double().numpy()
        assert (np.abs(got - want) <= (2 * 256 * total + np.abs(want)) * 2.0 ** -24).all()     # as mx_cases.py derives it
