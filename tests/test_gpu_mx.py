"""GPU parity of the layer operators against the CPU oracle (oracle/mx_oracle.py); bounds in mx_cases.py."""
import numpy as np
import pytest
import torch

from conftest import pkg
from mx_cases import (DTYPES, FORMATS, GATED, NORM, U, assert_mx, assert_near, bits, codes_of, f64, hidden, half_ulp,
                      small_integers)
from oracle import mx_oracle as ORACLE

pytestmark = pytest.mark.gpu
MX = pkg("mx")

INF, NAN = float("inf"), float("nan")


def fmt_of(q):
    return "mxfp8" if q.codes.dtype is torch.float8_e4m3fn else "mxfp4"


def assert_rounded(q, x, fmt):
    """Quantisation computes nothing that float32 does not hold: the oracle's values and exponents, bit for bit."""
    want, e = ORACLE.quantize(x, fmt)
    got, e_got = codes_of(q)
    assert fmt_of(q) == fmt and q.cols == x.shape[1]
    assert np.array_equal(e_got, e)
    assert np.array_equal(got, want, equal_nan=True)


# ---------------------------------------------------------------------------------------------- quantisation

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (1, 32), (5, 33), (2, 100), (4, 128), (257, 200), (3, 1481),
                                       (300, 2048), (2, 16390)])
def test_quantize(device, dtype, fmt, rows, cols):
    x = hidden(rows * 7 + cols, rows, cols, dtype)
    q = MX.quantize_mx_hip(x.to(device), fmt)
    assert_rounded(q, f64(x), fmt)
    for to in DTYPES:
        v = MX.dequantize_mx_hip(q, to)
        assert v.dtype is to and v.shape == (rows, cols)
        assert torch.equal(v.cpu(), torch.from_numpy(codes_of(q)[0][:, :cols]).to(torch.float32).to(to))


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_every_16_bit_pattern(device, fmt):
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
        lone = torch.zeros(2048, 32, 32, dtype=dtype)      # each pattern in a block with a smaller finite one
        lone[:, :, 5] = x.view(2048, 32)
        lone[:, :, 20] = (x.view(2048, 32).float() * 0.37).to(dtype)
        for y in (x.view(64, 1024), lone.view(2048, 1024)):
            assert_rounded(MX.quantize_mx_hip(y.to(device), fmt), f64(y), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_ties_and_ends(device, fmt):
    grid = np.sort(ORACLE.E2M1[:8] if fmt == "mxfp4" else ORACLE.E4M3[:127])
    near = np.concatenate([grid, (grid[1:] + grid[:-1]) / 2])
    near = np.concatenate([near, near * (1 - 2.0 ** -20), near * (1 + 2.0 ** -20)])
    near = np.concatenate([near, -near])
    most = 7.99 if fmt == "mxfp4" else 511.0
    x = np.zeros((5, -(-near.size // 31) * 32))
    for i in range(near.size):
        x[:, i // 31 * 32 + i % 31] = near[i]
    x[:, 31::32] = most
    x *= np.ldexp(1.0, np.array([0, 1, -30, 100, -140]))[:, None]     # the last: float32's subnormals
    y = torch.from_numpy(x).to(torch.float32)
    assert_rounded(MX.quantize_mx_hip(y.to(device), fmt), f64(y), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_non_finite_blocks(device, fmt):
    x = hidden(5, 6, 160, torch.float32)
    x[0, 3], x[1, 40], x[2, 159], x[3, 0], x[3, 31] = NAN, INF, -INF, INF, NAN
    x[4] = 0
    assert_rounded(MX.quantize_mx_hip(x.to(device), fmt), f64(x), fmt)
    q = MX.quantize_mx_hip(x.to(device), fmt)
    v = MX.dequantize_mx_hip(q, torch.float32).cpu()
    assert v[0, :32].isnan().all() and v[0, 32:].isfinite().all() and not v[4].any()


def test_quantize_views_rows_and_out(device):
    wide = hidden(6, 50, 700).to(device)
    x = wide[:, 33:533]                                  # rows at odd addresses
    idx = torch.tensor([49, 0, 7, 7, -1, 50, 3, 2 ** 40], device=device)
    for fmt in FORMATS:
        q = MX.quantize_mx_hip(x, fmt, rows=idx)
        want = np.full((8, 500), np.nan)
        for i, j in enumerate(idx.tolist()):
            if 0 <= j < 50:
                want[i] = f64(x[j])
        want[[4, 5, 7]] = np.nan
        assert_rounded(q, want, fmt)
        codes = torch.full((10, 512 if fmt == "mxfp8" else 256), 0x55, dtype=torch.uint8, device=device).view(q.codes.dtype)
        scales = torch.full((10, 32), 0x55, dtype=torch.uint8, device=device).view(q.scales.dtype)
        got = MX.quantize_mx_hip(x, fmt, rows=idx, out=(codes[1:9], scales[1:9, 8:24]))
        assert np.array_equal(bits(got.codes), bits(q.codes)) and np.array_equal(bits(got.scales), bits(q.scales))
        for t in (codes[0], codes[9], scales[0], scales[9], scales[:, :8], scales[:, 24:]):
            assert (bits(t) == 0x55).all()
    assert MX.quantize_mx_hip(x, rows=idx[:0]).codes.shape == (0, 256)
    assert MX.quantize_mx_hip(x[:0]).scales.shape == (0, 16)


# ---------------------------------------------------------------------------------------------- norm

def check_norm(x, w, device, residual=None, rows=None, formats=(None, *FORMATS), eps=1e-5, want_sum=True):
    """x, w, residual, rows on the CPU (rows of an index outside x are NaN)."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    if rows is not None:
        ok = (rows >= 0) & (rows < x.shape[0])
        h = torch.where(ok[:, None], h[rows.clamp(0, x.shape[0] - 1)], NAN)
    want = ORACLE.rms_norm(f64(h), f64(w), eps)
    put = lambda t: None if t is None else t.to(device)  # noqa: E731
    for fmt in formats:
        total = torch.full_like(h, 7.0, device=device) if want_sum else None
        got = MX.rms_norm_hip(put(x), put(w), eps, residual=put(residual), sum_out=total, rows=put(rows), format=fmt)
        if fmt is None:
            assert got.dtype is x.dtype
            assert_near(got, want, x.dtype, NORM)
        else:
            assert_mx(got, want, fmt, NORM)
        if total is not None:
            assert torch.equal(total.cpu().nan_to_num(1.5), h.nan_to_num(1.5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 7, 8, 64, 129, 200, 512, 513, 2048, 2049, 4096, 4104, 16384, 32768, 32769, 50003])
def test_norm_widths(device, dtype, cols):
    rows = 3 if cols > 4096 else 37
    x, r = hidden(cols, rows, cols, dtype), hidden(cols + 1, rows, cols, dtype)
    w = 1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(cols))
    check_norm(x, w.to(dtype), device, r)
    check_norm(x, w, device, want_sum=False)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 1000])
def test_norm_rows(device, rows):
    for cols in (24, 128, 1000):
        check_norm(hidden(rows, rows, cols), torch.ones(cols, dtype=torch.bfloat16), device, hidden(rows + 1, rows, cols))


def test_norm_picks_rows(device):
    idx = torch.tensor([9, 3, 3, 0, -1, 10, 2 ** 33, 5])
    for cols in (100, 2048, 40000):
        x, r = hidden(1, 10, cols), hidden(2, 10, cols)
        check_norm(x, torch.ones(cols), device, r, idx)
        check_norm(x, torch.ones(cols), device, None, idx, want_sum=False)
        check_norm(x, torch.ones(cols), device, r, torch.arange(10).repeat(30))


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_sizes_of_values(device, dtype):
    """Rows of zeros, of the largest and the least values, non-finite ones, and eps of zero."""
    big = float(torch.finfo(dtype).max) / 4
    least = float(torch.finfo(dtype).smallest_normal)
    x = hidden(3, 9, 640, torch.float32)
    x = x / x.abs().amax(1, keepdim=True)
    x[1], x[2], x[3], x[4] = 0, x[2] * big, x[3] * least, x[4] * least * 2.0 ** -6
    x[5, 10], x[6, 639], x[7, 0] = NAN, INF, -INF
    x = x.to(dtype)
    w = torch.randn(640, generator=torch.Generator().manual_seed(4)).to(dtype)
    for eps in (1e-5, 1e-30, 0.0):
        keep = torch.tensor([0, 2, 3, 5, 6, 7, 8]) if eps == 0.0 else torch.arange(9)
        check_norm(x[keep], w, device, eps=eps)
    zero = MX.rms_norm_hip(x[1:2].to(device), w.to(device), 0.0)     # 0 / 0
    assert zero.isnan().all()


def test_norm_heads_on_views(device):
    for dtype in DTYPES:
        for tokens, heads, d in ((70, 5, 128), (1, 40, 64), (33, 3, 100), (2, 2, 4096)):
            qkv = hidden(d, tokens, (heads + 3) * d, dtype)
            x = qkv[:, d:(heads + 1) * d].view(tokens, heads, d)
            w = 1 + 0.1 * torch.randn(d, generator=torch.Generator().manual_seed(9))
            want = ORACLE.rms_norm(f64(x), f64(w), 1e-6)
            dev = qkv.to(device)
            xd = dev[:, d:(heads + 1) * d].view(tokens, heads, d)
            assert_near(MX.rms_norm_hip(xd, w.to(device), 1e-6), want, dtype, NORM)
            MX.rms_norm_hip(xd, w.to(device), 1e-6, out=xd)                     # in place, the other heads untouched
            assert_near(xd, want, dtype, NORM)
            assert torch.equal(dev[:, :d].cpu(), qkv[:, :d]) and torch.equal(dev[:, (heads + 1) * d:].cpu(), qkv[:, (heads + 1) * d:])


@pytest.mark.parametrize("cols", [130, 4096, 40000])
def test_norm_in_place(device, cols):
    x, r = hidden(1, 20, cols), hidden(2, 20, cols)
    w = torch.ones(cols, dtype=torch.bfloat16, device=device)
    h = (x.float() + r.float()).to(x.dtype)
    want = ORACLE.rms_norm(f64(h), np.ones(cols), 1e-5)
    for swap in (False, True):
        xd, rd = x.to(device), r.to(device)
        s, o = (xd, rd) if swap else (rd, xd)
        got = MX.rms_norm_hip(xd, w, 1e-5, residual=rd, sum_out=s, out=o)
        assert got is o and torch.equal(s.cpu(), h)
        assert_near(o, want, x.dtype, NORM)


def test_overlapping_results_are_refused(device):
    x = torch.zeros(8, 256, device=device)
    w, idx = torch.ones(256, device=device), torch.arange(8, device=device)
    both = torch.zeros(8, 512, device=device)
    for src, kw in ((x, dict(out=x, rows=idx)), (x, dict(sum_out=x, rows=idx)), (x, dict(out=x, residual=x, sum_out=x)),
                    (both[:, :256], dict(out=both[:, 1:257])), (both[:4, :256], dict(out=both[1:5, :256]))):
        with pytest.raises(MX.MxError, match="overlap"):
            MX.rms_norm_hip(src, w, 1e-5, **kw)
    with pytest.raises(MX.MxError, match="rows overlap"):
        MX.rms_norm_hip(x, w, 1e-5, out=torch.zeros(256, device=device).expand(8, 256))
    with pytest.raises(MX.MxError, match="overlap"):
        MX.silu_mul_hip(both[:, :256], both[:, 256:], out=both[:, 128:384])
    room = torch.zeros(1 << 16, dtype=torch.uint8, device=device)
    codes, scales = room[1024:1024 + 4096].view(torch.float4_e2m1fn_x2).view(8, 512), room[:256].view(torch.float8_e8m0fnu).view(8, 32)
    out = room[4096:4096 + 16384].view(torch.bfloat16).view(8, 1024)
    with pytest.raises(MX.MxError, match="overlap"):
        MX.dequantize_mx_hip((codes, scales), out=out)
    with pytest.raises(MX.MxError, match="overlap"):
        MX.mx_linear_hip((codes, scales), (codes, scales), out=out[:, :8])
    MX.rms_norm_hip(both[:, :256], w, 1e-5, out=both[:, 256:])               # beside each other
    MX.silu_mul_hip(both[:, :256], both[:, 256:], out=both[:, :256])


# ---------------------------------------------------------------------------------------------- gated

def check_gated(g, u, device, formats=(None, *FORMATS)):
    want = ORACLE.silu_mul(f64(g), f64(u))
    floor = 2.0 ** -149 * (1 + np.abs(f64(g))) * (1 + np.abs(f64(u)))
    floor = np.where(np.isfinite(floor), floor, 0.0)
    for fmt in formats:
        got = MX.silu_mul_hip(g.to(device), u.to(device), format=fmt)
        if fmt is None:
            assert_near(got, want, g.dtype, GATED, floor)
        else:
            assert_mx(got, want, fmt, GATED, floor)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8192), (5, 33), (64, 128), (300, 777), (3, 14336), (1025, 40)])
def test_silu_mul(device, dtype, rows, cols):
    both = hidden(rows + cols, rows, 2 * cols, dtype, 0.5)
    check_gated(both[:, :cols], both[:, cols:], device)
    dev = both.to(device)
    got = MX.silu_mul_hip(dev[:, :cols], dev[:, cols:])
    assert torch.equal(got, MX.silu_mul_hip(dev[:, :cols].contiguous(), dev[:, cols:].contiguous()))
    assert MX.silu_mul_hip(dev[:, :cols], dev[:, cols:], out=dev[:, cols:]).data_ptr() == dev[:, cols:].data_ptr()
    assert torch.equal(dev[:, cols:], got) and torch.equal(dev[:, :cols].cpu(), both[:, :cols])


def test_silu_mul_far_gates(device):
    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20, -20, 87, -87, -88.5, -95, -103, -104, 1000, -1000, 3e38, -3e38, INF, NAN])
    u = torch.tensor([1.0, -2.0, 1e10, 1e20, 3e38, INF])
    g, u = g.repeat_interleave(len(u))[None], u.repeat(len(g))[None]
    far = (g > -1e30) & ~(g.isinf() | g.isnan()) & ~u.isinf()
    check_gated(g[far][None], u[far][None], device, (None,))
    got = MX.silu_mul_hip(torch.tensor([[INF, -INF, NAN, 1.0, -1.0]], device=device), torch.tensor([[2.0, 2.0, 2.0, INF, INF]], device=device))
    assert got[0, 0] == INF and got[0, 1:3].isnan().all() and got[0, 3] == INF and got[0, 4] == -INF


# ---------------------------------------------------------------------------------------------- products

def check_exact(m, n, cols, fmt, device, dtype=torch.float32, seed=0, **kw):
    """Whole multiples that float32 adds exactly in any order: the result is the formula's, rounded once."""
    x, xv = small_integers(seed + m, m, cols, fmt, device)
    w, wv = small_integers(seed + n + 1, n, cols, "mxfp4", device)
    print(f"linear: m {m} n {n} cols {cols} {fmt} {dtype}", flush=True)
    got = MX.mx_linear_hip(x, w, dtype=dtype, **kw)
    want = torch.from_numpy(xv @ wv.T).to(torch.float32).to(dtype)
    assert got.shape == (m, n) and torch.equal(got.cpu(), want)
    return x, w, want


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 48, 64, 65, 100, 128, 129, 200, 256, 257, 513])
def test_linear_rows(device, fmt, m):
    for n, cols in ((1, 32), (15, 160), (257, 384), (520, 1000)):
        check_exact(m, n, cols, fmt, device)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n", [1, 2, 16, 31, 64, 100, 128, 255, 256, 1000, 4099])
def test_linear_columns(device, fmt, n):
    for m, cols in ((1, 2048), (3, 128), (40, 640), (130, 256), (300, 544)):
        check_exact(m, n, cols, fmt, device, torch.bfloat16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("cols", [1, 32, 128, 129, 256, 512, 640, 896, 1024, 1152, 2048, 4096, 5000, 16384])
def test_linear_widths(device, fmt, cols):
    for m, n in ((1, 48), (20, 300), (64, 96), (150, 130), (260, 270)):
        check_exact(m, n, cols, fmt, device, torch.float16 if cols < 1000 else torch.float32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,cols", [(1, 8192, 2048), (5, 128256, 128), (64, 20000, 2048), (700, 2048, 1024), (2049, 700, 512),
                                      (1100, 3000, 768)])
def test_linear_large(device, fmt, m, n, cols):
    check_exact(m, n, cols, fmt, device)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_of_quantized_rows(device, dtype, fmt):
    """Real values and scales of many sizes, to the bound of a sum in float32."""
    for m, n, cols in ((1, 300, 1000), (7, 513, 4096), (70, 200, 2048), (300, 400, 1500)):
        x = MX.quantize_mx_hip(hidden(m, m, cols).to(device), fmt)
        w = MX.quantize_mx_hip((hidden(n, n, cols) * 0.02).to(device), "mxfp4")
        want, total = ORACLE.linear(codes_of(x)[0], codes_of(w)[0])
        assert_near(MX.mx_linear_hip(x, w, dtype=dtype), want, dtype, 0.0, 2 * x.codes.shape[1] * U * total + np.abs(want) * U)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_non_finite_rows(device, m):
    for fmt in FORMATS:
        xh, wh = hidden(m, m, 500, torch.float32), hidden(3, 90, 500, torch.float32) * 0.1
        xh[m // 2, 400], wh[17, 3], wh[89, 499] = INF, NAN, -INF
        x, w = MX.quantize_mx_hip(xh.to(device), fmt), MX.quantize_mx_hip(wh.to(device), "mxfp4")
        nan = np.zeros((m, 90), dtype=bool)
        nan[m // 2], nan[:, [17, 89]] = True, True
        got = MX.mx_linear_hip(x, w, dtype=torch.float32).cpu()
        assert np.array_equal(got.isnan().numpy(), nan)
        want, total = ORACLE.linear(np.nan_to_num(codes_of(x)[0]), np.nan_to_num(codes_of(w)[0]))
        assert (np.abs(got.numpy()[~nan] - want[~nan]) <= 2 * 512 * U * total[~nan] + U * np.abs(want[~nan])).all()


def test_linear_scales_at_the_ends(device):
    for e in (-60, -100, 60):
        for m in (1, 40, 200):
            x, xv = small_integers(1, m, 256, "mxfp8", device)
            w, wv = small_integers(2, 50, 256, "mxfp4", device)
            s = (x.scales.view(torch.uint8).int() + e).to(torch.uint8).view(torch.float8_e8m0fnu)
            t = (w.scales.view(torch.uint8).int() - e).to(torch.uint8).view(torch.float8_e8m0fnu)
            assert torch.equal(MX.mx_linear_hip((x.codes, s), (w.codes, t), dtype=torch.float32).cpu().double(), torch.from_numpy(xv @ wv.T))


@pytest.mark.parametrize("m,n", [(1, 64), (40, 90), (64, 25600), (128, 25600), (200, 25600)])
def test_linear_large_and_small_products_together(device, m, n):
    """Eight neighbours from e4m3's smallest value to its largest: their float32 sum is exact (magnitudes under 448 * 4 * 8 <
    2^14, whole multiples of 2^-9 / 2), and a 16-bit result loses at most 2^-13 of the largest product for each other one."""
    gen = torch.Generator().manual_seed(m)
    xc = torch.zeros(m, 128, dtype=torch.uint8)
    for i in range(m):
        some = torch.randint(0, 127, (8,), generator=gen) + 128 * torch.randint(0, 2, (8,), generator=gen)
        some[i % 8], some[(i + 3) % 8] = 126, 1                                   # 448 and 2^-9
        xc[i, 8 * (i % 16):8 * (i % 16) + 8] = some.to(torch.uint8)
    nibbles = torch.randint(0, 7, (n, 128), generator=gen) + 8 * torch.randint(0, 2, (n, 128), generator=gen)
    value = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
    xv, wv = xc.view(torch.float8_e4m3fn).double(), value[nibbles]
    one = lambda rows: torch.full((rows, 4), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu).to(device)
    x = (xc.view(torch.float8_e4m3fn).to(device), one(m))
    w = ((nibbles[:, 0::2] | nibbles[:, 1::2] << 4).to(torch.uint8).view(torch.float4_e2m1fn_x2).to(device), one(n))
    want = xv @ wv.T
    assert torch.equal(MX.mx_linear_hip(x, w, dtype=torch.float32).cpu().double(), want)
    largest = torch.full((m, 1), 448.0 * 4, dtype=torch.float64)
    for dtype in (torch.bfloat16, torch.float16):
        got = MX.mx_linear_hip(x, w, dtype=dtype).cpu().double()
        lost = 7 * 2.0 ** -13 * largest
        assert ((got - want).abs() <= lost + (want.abs() + lost) * torch.finfo(dtype).eps / 2).all()


@pytest.mark.parametrize("m", [3, 33, 140])
def test_linear_strided_operands_and_out(device, m):
    x, w, want = check_exact(m, 200, 384, "mxfp8", device, torch.bfloat16)
    big = torch.full((m + 2, 333), 9.0, dtype=torch.bfloat16, device=device)      # rows at odd addresses
    got = MX.mx_linear_hip(x, w, out=big[1:m + 1, 101:301])
    assert got.data_ptr() == big[1:, 101:].data_ptr()
    assert torch.equal(big[1:m + 1, 101:301].cpu(), want)
    big[1:m + 1, 101:301] = 9.0
    assert (big == 9.0).all()
    wide = torch.zeros(200, 512, dtype=torch.uint8, device=device)                # a weight's rows within wider ones
    wide[:, 64:256] = w.codes.view(torch.uint8)
    tall = torch.zeros(400, 12, dtype=torch.uint8, device=device)
    tall[::2] = w.scales.view(torch.uint8)
    strided = (wide[:, 64:256].view(w.codes.dtype), tall[::2].view(w.scales.dtype))
    assert torch.equal(MX.mx_linear_hip(x, strided).cpu(), want)
    some = MX.MxTensor(w.codes[50:60], w.scales[50:60], 384)
    assert torch.equal(MX.mx_linear_hip(x, some).cpu(), want[:, 50:60])
    assert MX.mx_linear_hip((x.codes[:0], x.scales[:0]), w).shape == (0, 200)
    assert MX.mx_linear_hip(x, (w.codes[:0], w.scales[:0])).shape == (m, 0)


def test_linear_rows_do_not_depend_on_the_batch(device):
    """A row's result is the same bits in every batch of one kernel, and run twice."""
    w = MX.quantize_mx_hip((hidden(1, 1000, 2048) * 0.02).to(device), "mxfp4")
    x = MX.quantize_mx_hip(hidden(2, 600, 2048).to(device), "mxfp8")
    for lo, hi in ((0, 600), (100, 130)):
        part = MX.MxTensor(x.codes[lo:hi], x.scales[lo:hi], 2048)
        assert torch.equal(MX.mx_linear_hip(part, w, dtype=torch.float32), MX.mx_linear_hip(part, w, dtype=torch.float32))


# ---------------------------------------------------------------------------------------------- far offsets

def test_rows_past_32_bits(device):
    """Matrices of more than 2^32 bytes: the last rows are those of a call on them alone."""
    n, cols = 70000, 65536
    x = torch.zeros(n, cols, dtype=torch.bfloat16, device=device)
    tail = hidden(1, 300, cols).to(device)
    x[-300:] = tail
    w = torch.ones(cols, dtype=torch.bfloat16, device=device)
    q = MX.quantize_mx_hip(x, "mxfp8")
    want = MX.quantize_mx_hip(tail, "mxfp8")
    assert torch.equal(q.codes[-300:].view(torch.uint8), want.codes.view(torch.uint8))
    assert torch.equal(q.scales[-300:].view(torch.uint8), want.scales.view(torch.uint8))
    y = MX.dequantize_mx_hip(q, torch.bfloat16)
    assert torch.equal(y[-300:], MX.dequantize_mx_hip(want, torch.bfloat16)) and not y[:100].any()
    del y
    assert torch.equal(MX.rms_norm_hip(x, w, 1e-5, rows=torch.arange(n - 300, n, device=device)), MX.rms_norm_hip(tail, w, 1e-5))
    out = MX.silu_mul_hip(x, x, out=x)
    assert torch.equal(out[-300:], MX.silu_mul_hip(tail, tail))
    # products: x of over 2^32 bytes times a few rows, and the other way about
    few, _ = small_integers(2, 40, cols, "mxfp4", device)
    got = MX.mx_linear_hip(q, few)
    part = MX.MxTensor(q.codes[-300:].clone(), q.scales[-300:].clone(), cols)
    assert torch.equal(got[-300:].isnan(), torch.zeros_like(got[-300:], dtype=torch.bool))
    # every tile adds the columns in their order, 128 at a time: the same sums, the same bits.  (A bound relative to a float32
    # result would not hold: that one keeps what a 16-bit one leaves out of an octet, up to 7 2^-13 of the sum of magnitudes,
    # and a result may be as small as it likes beside that sum.)
    assert torch.equal(got[-300:], MX.mx_linear_hip(part, few))
    del q, got, x, out
    long = torch.randint(0, 256, (140000, cols // 2), dtype=torch.uint8, device=device).view(torch.float4_e2m1fn_x2)
    scales = torch.full((140000, cols // 32), 120, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
    v, _ = small_integers(3, 3, cols, "mxfp8", device)
    got = MX.mx_linear_hip(v, (long, scales), dtype=torch.float32)
    assert torch.equal(got[:, -50:], MX.mx_linear_hip(v, (long[-50:].clone(), scales[-50:].clone()), dtype=torch.float32))


# ---------------------------------------------------------------------------------------------- streams, graphs, together

def layer_inputs(device, tokens, hidden_size=512, heads=8, kv=2, d=64, inter=768, vocab=3000):
    g = torch.Generator().manual_seed(tokens)
    mat = lambda n, k: MX.quantize_mx_hip((torch.randn(n, k, generator=g) / k ** 0.5).to(torch.bfloat16).to(device), "mxfp4")  # noqa: E731
    ones = lambda: (1 + 0.1 * torch.randn(hidden_size, generator=g)).to(torch.bfloat16).to(device)  # noqa: E731
    return dict(x=hidden(tokens, tokens, hidden_size).to(device), r=hidden(tokens + 1, tokens, hidden_size).to(device),
                qkv=mat((heads + 2 * kv) * d, hidden_size), o=mat(hidden_size, heads * d), up=mat(2 * inter, hidden_size),
                down=mat(hidden_size, inter), head=mat(vocab, hidden_size), n1=ones(), n2=ones(), n3=ones(), heads=heads, kv=kv, d=d,
                inter=inter)


def run_layer(p, cache, batch, sample, seen=None):
    """One decoder layer and the sampled rows' logits, through the entry points of all modules."""
    KV, PA = pkg("kv_cache"), pkg("paged_attention")
    keep = (lambda name, *v: seen.append((name, *v[:-1], v[-1].clone() if isinstance(v[-1], torch.Tensor) else v[-1]))) \
        if seen is not None else (lambda *a: None)
    heads, kv, d = p["heads"], p["kv"], p["d"]
    tables, lens, starts, qlens, inv = batch
    r = torch.empty_like(p["r"])
    h = MX.rms_norm_hip(p["x"], p["n1"], 1e-5, residual=p["r"], sum_out=r, format="mxfp8")
    keep("norm", p["x"], p["r"], p["n1"], h)
    qkv = MX.mx_linear_hip(h, p["qkv"])
    keep("linear", h, p["qkv"], qkv)
    n = qkv.shape[0]
    q, k, v = (t.view(n, -1, d) for t in qkv.split((heads * d, kv * d, kv * d), dim=1))
    KV.store_kv_hip(k, v, *cache, tables, lens, starts, qlens, 16, query=q, inv_freq=inv, out=q)
    a = PA.paged_attention_hip(q, *cache, tables, lens, starts, qlens, d ** -0.5, 16, max_query_len=1, max_seq_len=64)
    a8 = MX.quantize_mx_hip(a.reshape(n, heads * d), "mxfp8")
    x = MX.mx_linear_hip(a8, p["o"])
    keep("linear", a8, p["o"], x)
    r2 = torch.empty_like(r)
    h = MX.rms_norm_hip(x, p["n2"], 1e-5, residual=r, sum_out=r2, format="mxfp8")
    keep("norm", x, r, p["n2"], h)
    both = MX.mx_linear_hip(h, p["up"])
    act = MX.silu_mul_hip(both[:, :p["inter"]], both[:, p["inter"]:], format="mxfp8")
    keep("gated", both, act)
    x = MX.mx_linear_hip(act, p["down"])
    keep("linear", act, p["down"], x)
    last = MX.rms_norm_hip(x, p["n3"], 1e-5, residual=r2, rows=sample, format="mxfp8")
    logits = MX.mx_linear_hip(last, p["head"], dtype=torch.float32)
    keep("linear", last, p["head"], logits)
    return logits


def decode_batch(device, tokens):
    tables = torch.arange(1, 1 + 4 * tokens, dtype=torch.int32, device=device).view(tokens, 4)
    lens = torch.arange(20, 20 + tokens, dtype=torch.int32, device=device) % 60 + 1
    starts = torch.arange(tokens + 1, dtype=torch.int32, device=device)
    inv = (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float().to(device)
    cache = [torch.randn(1 + 4 * tokens, 16, 2, 64, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(device) for i in (1, 2)]
    return cache, (tables, lens, starts, torch.ones_like(lens), inv)


@pytest.mark.parametrize("tokens", [3, 70])
def test_a_layer_and_its_logits(device, tokens):
    p = layer_inputs(device, tokens)
    cache, batch = decode_batch(device, tokens)
    sample = torch.arange(0, tokens, 2, device=device)
    seen = []
    logits = run_layer(p, cache, batch, sample, seen)
    for name, *t in seen:
        if name == "norm":
            x, r, w, out = t
            h = (x.float() + r.float()).to(x.dtype)
            assert_mx(out, ORACLE.rms_norm(f64(h), f64(w), 1e-5), "mxfp8", NORM)
        elif name == "gated":
            both, out = f64(t[0]), t[1]
            assert_mx(out, ORACLE.silu_mul(both[:, :p["inter"]], both[:, p["inter"]:]), "mxfp8", GATED)
        else:
            x, w, out = t
            want, total = ORACLE.linear(codes_of(x)[0], codes_of(w)[0])
            assert_near(out, want, out.dtype, 0.0, 2 * x.codes.shape[1] * U * total + np.abs(want) * U)
    S = pkg()
    params = [S.SamplingParams(temperature=0.0)] * len(sample)
    ids = S.Sampler(device).sample(logits, params, [[]] * len(sample))
    assert ids.tolist() == logits.argmax(1).tolist()


def test_a_layer_captured_and_replayed(device):
    p = layer_inputs(device, 8)
    cache, batch = decode_batch(device, 8)
    sample = torch.tensor([7, 0, 3], device=device)
    run_layer(p, cache, batch, sample)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run_layer(p, cache, batch, sample)
    for i in range(4):
        p["x"].copy_(hidden(50 + i, 8, 512))
        p["r"].copy_(hidden(60 + i, 8, 512))
        sample.copy_(torch.tensor([i, 7 - i, 2]))
        got.fill_(-1.0)
        g.replay()
        torch.cuda.synchronize()
        first = got.clone()
        want = run_layer(p, cache, batch, sample)
        assert torch.equal(first, want)
        g.replay()
        assert torch.equal(got, want)


def test_calls_on_two_streams(device):
    """Calls keep nothing between them: two streams' calls do not meet, and a call runs on the stream that it is given."""
    w = MX.quantize_mx_hip((hidden(1, 4096, 2048) * 0.02).to(device), "mxfp4")
    xs = [hidden(s, m, 2048).to(device) for s, m in ((2, 1), (3, 64), (4, 300))]
    ones = torch.ones(2048, dtype=torch.bfloat16, device=device)

    def chain(x, **kw):
        h = MX.rms_norm_hip(x, ones, 1e-5, format="mxfp8", **kw)
        y = MX.mx_linear_hip(h, w, **kw)
        return MX.dequantize_mx_hip(MX.quantize_mx_hip(MX.silu_mul_hip(y[:, :2048], y[:, 2048:], **kw), "mxfp4", **kw), **kw)

    want = [chain(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = [chain(x, stream=s if i else s.cuda_stream) for i, (x, s) in enumerate(zip(xs, streams))]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    slow = torch.cuda.Stream()
    with torch.cuda.stream(slow):
        torch.cuda._sleep(200_000_000)
        x = xs[1] + 0
    got = chain(x, stream=slow)       # behind the sleep
    slow.synchronize()
    assert torch.equal(got, want[1])
    assert torch.equal(chain(xs[0], stream=0), want[0])
