"""silu(gate) * up in float32, to the roundings that it cannot do without.

With u = 2^-24: the exponential within 2 u (the device library's 1 ulp), of which a gate below zero sees less than the whole
(e / (1 + e) of it) and one above less than half; 1 + e, the quotient and the product by up round once each: 5 u.  Far gates
round gate * e in place of 1 + e.  Below the normal numbers 2^-149 of the exponential is lost, times |gate up|."""
import numpy as np
import pytest
import torch

from conftest import pkg
from mx_cases import U, f64
from oracle import mx_oracle as ORACLE

pytestmark = pytest.mark.gpu
MX = pkg("mx")


def check(gate, up, device):
    want = ORACLE.silu_mul(f64(gate), f64(up))
    got = f64(MX.silu_mul_hip(gate.to(device), up.to(device)))
    floor = 2.0 ** -149 * (1 + np.abs(f64(gate))) * (1 + np.abs(f64(up)))
    off = np.abs(got - want) - floor
    assert (off <= 5 * U * np.abs(want)).all(), (off / np.abs(want)).max() / U


def test_float32_gates(device):
    g = torch.Generator().manual_seed(7)
    check(torch.randn(1024, 8192, generator=g) * 3, torch.randn(1024, 8192, generator=g), device)


def test_float32_gates_of_every_size(device):
    g = torch.Generator().manual_seed(8)
    gate = torch.cat([torch.linspace(-104, 104, 100001), torch.randn(65536, generator=g).sign() * torch.logspace(-40, 2, 65536),
                      torch.tensor([-80.0, -80.00001, -79.99999, -88.7, -87.3, -103.9, 0.0, -0.0])])
    for size in (1.0, 1e-30, 1e30):
        check(gate[None], torch.full_like(gate, size)[None], device)


def test_float32_rows_at_any_alignment_and_neighbours_at_the_ends(device):
    """A chunk of eight that holds infinities, NaN and far gates beside near ones: each value is its own."""
    inf, nan = float("inf"), float("nan")
    gate = torch.tensor([1.0, -1.0, inf, -inf, nan, -100.0, 100.0, 0.5, -3.0, 2.0, -90.0])
    for start in range(4):
        got = MX.silu_mul_hip(gate[None, start:].to(device), torch.full((1, 11 - start), 2.0, device=device))[0].cpu().double()
        want = gate[start:].double()
        want = torch.nn.functional.silu(want) * 2
        want[torch.isneginf(gate[start:])] = nan
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[want == inf], want[want == inf])
        fine = want.isfinite()
        assert ((got - want)[fine].abs() <= 5 * U * want[fine].abs() + 2.0 ** -140).all()
