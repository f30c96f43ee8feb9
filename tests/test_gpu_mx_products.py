"""Products of MX rows on the GPU: every kernel that a size can take, its loops and its tails, results of each type.

``mx_cases.py`` says how the bounds of sums come about.  Products are whole for every type of result: a 16-bit result is the
float32 one rounded once."""
import pytest
import torch

from conftest import pkg
from mx_cases import hidden
from mx_kernels import SIZES, kernel_of, kernels_of, widths

pytestmark = pytest.mark.gpu
MX = pkg("mx")

E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)

# (rows, outputs, columns), one or more for each kernel of 8-bit rows
KERNELS_8 = [(1, 40, 256), (16, 90, 2176), (16, 16384, 384), (40, 70, 640), (17, 8100, 384), (50, 8300, 640), (64, 16500, 256),
             (60, 32900, 384), (70, 51300, 384), (300, 17000, 640)]


@pytest.mark.parametrize("m,n,k", KERNELS_8)
def test_large_products_that_cancel_leave_the_small_ones(device, m, n, k):
    """Of eight neighbours two are 448 and -448 times one weight, the others below 2: the sum is the others', whole multiples
    of 2^-10 below 2^13, which float32 adds exactly in any order."""
    gen = torch.Generator().manual_seed(m)
    xc = torch.randint(0, 64, (m, k // 8, 8), generator=gen) + 128 * torch.randint(0, 2, (m, k // 8, 8), generator=gen)
    xc[..., 2], xc[..., 5] = 0x7e, 0xfe
    xc[..., 2:6:3] ^= 128 * torch.randint(0, 2, (m, k // 8, 1), generator=gen)
    xc = xc.view(m, k).to(torch.uint8)
    nibbles = torch.randint(0, 16, (n, k // 8, 8), generator=gen)
    nibbles[..., 5] = nibbles[..., 2]
    nibbles = nibbles.view(n, k)
    one = lambda rows: torch.full((rows, k // 32), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu).to(device)  # noqa: E731
    x = (xc.view(torch.float8_e4m3fn).to(device), one(m))
    w = ((nibbles[:, 0::2] | nibbles[:, 1::2] << 4).to(torch.uint8).view(torch.float4_e2m1fn_x2).to(device), one(n))
    # float32 on the host is exact here as well, but not in every order of the large ones: without them
    small = xc.view(torch.float8_e4m3fn).float()
    small[small.abs() == 448] = 0
    want = small @ E2M1.float()[nibbles].T
    print(f"cancel: m {m} n {n} k {k}", flush=True)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        got = MX.mx_linear_hip(x, w, dtype=dtype)
        assert torch.equal(got.cpu(), want.to(dtype)), dtype


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("m,n,k", KERNELS_8)
def test_16_bit_results_are_the_float32_ones_rounded(device, fmt, m, n, k):
    x = MX.quantize_mx_hip(hidden(m, m, k).to(device), fmt)
    w = MX.quantize_mx_hip((hidden(n, n, k) * 0.02).to(device), "mxfp4")
    full = MX.mx_linear_hip(x, w, dtype=torch.float32)
    for dtype in (torch.bfloat16, torch.float16):
        assert torch.equal(MX.mx_linear_hip(x, w, dtype=dtype), full.to(dtype)), dtype


def whole_numbers(seed, rows, k, fmt, device):
    """MX rows on the device whose values are whole multiples of 2^-3, below 2^6, and the values in float64: their products'
    sums, of either sign, stay far below the 2^24 multiples of 2^-6 that float32 adds exactly in any order."""
    gen = torch.Generator(device=device).manual_seed(seed)
    pick = lambda lo, hi, *size: torch.randint(lo, hi, size, generator=gen, device=device)  # noqa: E731
    scales = pick(125, 130, rows, k // 32).to(torch.uint8)
    if fmt == "mxfp4":
        codes = pick(0, 256, rows, k // 2).to(torch.uint8)
        c = codes.long()
        v = E2M1.to(device)[torch.stack([c & 15, c >> 4], -1).view(rows, k)]
        codes = codes.view(torch.float4_e2m1fn_x2)
    else:
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 5, 6, 7, 8, -0.5, -1, -1.5, -2, -3, -4, -5, -6, -7, -8], device=device)
        v = grid[pick(0, len(grid), rows, k)]
        codes, v = v.to(torch.float8_e4m3fn), v.double()
    v = v.view(rows, -1, 32) * torch.exp2(scales.double() - 127)[..., None]
    return (codes, scales.view(torch.float8_e8m0fnu)), v.view(rows, k)


@pytest.mark.parametrize("fmt,m,n", SIZES)
def test_every_kernel_over_its_loop_and_tail(device, fmt, m, n):
    """The formula's result, rounded once, at widths of one stage up to more than two rounds of the kernel's loop."""
    for kernel in kernels_of(fmt, m, n):
        for k in widths(kernel):
            assert kernel_of(fmt, m, n, k) == kernel
            x, xv = whole_numbers(m + k, m, k, fmt, device)
            w, wv = whole_numbers(n + k + 1, n, k, "mxfp4", device)
            want = xv @ wv.T
            print(f"linear: m {m} n {n} k {k} {fmt} {kernel}", flush=True)
            assert want.abs().max() < 2 ** 15
            for dtype in (torch.bfloat16, torch.float16, torch.float32):
                got = MX.mx_linear_hip(x, w, dtype=dtype)
                assert torch.equal(got, want.float().to(dtype)), (kernel, k, dtype, (got.double() - want).abs().max().item())


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_a_row_gives_the_same_bits_in_every_batch_of_tiles(device, fmt):
    """All tiles add the columns in their order, so a row's results are the same bits wherever it stands and whichever tile
    its batch takes.  (few_kernel, up to 16 rows, cuts the columns over its waves.)"""
    seen = set()
    for n, k in ((1000, 2048), (9000, 1152), (26000, 640)):
        w = MX.quantize_mx_hip((hidden(n, n, k) * 0.02).to(device), "mxfp4")
        x = MX.quantize_mx_hip(hidden(k, 1400, k).to(device), fmt)
        for dtype in (torch.float32, torch.bfloat16):
            full = MX.mx_linear_hip(x, w, dtype=dtype)
            for lo, hi in ((0, 1400), (100, 130), (3, 67), (255, 455), (700, 1399), (1383, 1400)):
                part = MX.MxTensor(x.codes[lo:hi], x.scales[lo:hi], k)
                seen.add(kernel_of(fmt, hi - lo, n, k))
                assert torch.equal(MX.mx_linear_hip(part, w, dtype=dtype), full[lo:hi]), (n, lo, hi)
    assert len(seen) >= 4 and all(name == "tile" for name, *_ in seen)


@pytest.mark.parametrize("m,n,k", KERNELS_8)
def test_nan_codes_and_scales_stay_in_their_row_and_column(device, m, n, k):
    """e4m3's NaN codes of either sign, and scales of 255, on rows of x and of the weight; every other result is whole."""
    x, xv = whole_numbers(m, m, k, "mxfp8", device)
    w, wv = whole_numbers(n, n, k, "mxfp4", device)
    codes = x[0].view(torch.uint8)
    codes[m - 1, 7], codes[0, k - 1] = 0x7f, 0xff
    for row, block in ((0, 1), (n - 1, k // 32 - 1)):
        w[1].view(torch.uint8)[row, block] = 255
    nan = torch.zeros(m, n, dtype=torch.bool, device=device)
    nan[[0, m - 1]], nan[:, [0, n - 1]] = True, True
    got = MX.mx_linear_hip(x, w, dtype=torch.float32)
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan], (xv @ wv.T).float()[~nan])


@pytest.mark.parametrize("m,n,k", KERNELS_8)
def test_halves_at_their_ends_are_whole(device, m, n, k):
    """The widest octets of either half: 448 or 1.875 times 6 beside the half's least codes (2.25 above, 2^-9 below) times 0.5.
    Whole multiples of 2^-3 or 2^-10 whose sums stay below 2^24 of them."""
    gen = torch.Generator().manual_seed(n)
    for most, least, other in ((0x7e, 0x41, 0x47), (0x3f, 0x01, 0x0f)):
        xc = torch.where(torch.rand(m, k // 8, 8, generator=gen) < 0.5, least, other)
        xc[..., 3] = most
        xc = (xc + 128 * torch.randint(0, 2, xc.shape, generator=gen)).view(m, k).to(torch.uint8)
        nibbles = torch.full((n, k // 8, 8), 1)
        nibbles[..., 3] = 7
        nibbles = (nibbles + 8 * torch.randint(0, 2, nibbles.shape, generator=gen)).view(n, k)
        one = lambda rows: torch.full((rows, k // 32), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu).to(device)  # noqa: E731
        x = (xc.view(torch.float8_e4m3fn).to(device), one(m))
        w = ((nibbles[:, 0::2] | nibbles[:, 1::2] << 4).to(torch.uint8).view(torch.float4_e2m1fn_x2).to(device), one(n))
        want = x[0].double() @ E2M1[nibbles].to(device).T
        print(f"ends: m {m} n {n} k {k} most {most}", flush=True)
        for dtype in (torch.float32, torch.bfloat16):
            assert torch.equal(MX.mx_linear_hip(x, w, dtype=dtype), want.float().to(dtype)), (most, dtype)
