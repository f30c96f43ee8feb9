"""Products of MX rows on the GPU: every kernel that a size can take, its loops and its tails, results of each type.

``mx_cases.py`` says how the bounds of sums come about.  Products are whole for every type of result: a 16-bit result is the
float32 one rounded once."""
import pytest
import torch

from conftest import pkg
from mx_cases import hidden

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
