"""Arguments that the layer operators' calls take or refuse before any launch."""
import pytest
import torch

from conftest import pkg

MX = pkg("mx")


def test_rows_of_one_value_have_any_stride_along_the_row():
    """A result of one column in a column of something wider: no stride leads along such a row.  (What refuses these calls
    is the last check, that for the device.)"""
    x, w = torch.zeros(4, 1), torch.ones(1)
    out = torch.zeros(1, 4).t()
    assert out.shape == (4, 1) and out.stride() == (1, 4)
    with pytest.raises(MX.MxError, match="device tensors"):
        MX.rms_norm_hip(x, w, 1e-5, out=out, sum_out=torch.zeros(1, 4).t())
    with pytest.raises(MX.MxError, match="device tensors"):
        MX.silu_mul_hip(out, out, out=torch.zeros(1, 4).t())
    with pytest.raises(MX.MxError, match="unit stride"):
        MX.rms_norm_hip(torch.zeros(4, 2), torch.ones(2), 1e-5, out=torch.zeros(2, 4).t())


@pytest.mark.gpu
def test_rows_of_one_value_into_a_wider_tensor(device):
    x = torch.tensor([[3.0], [-2.0], [0.5], [7.0]], device=device)
    room = torch.full((2, 4), 9.0, device=device)
    got = MX.rms_norm_hip(x, torch.full((1,), 2.0, device=device), 0.0, out=room.t()[:, :1])
    assert got.data_ptr() == room.data_ptr() and torch.equal(room.cpu(), torch.tensor([[2.0, -2, 2, 2], [9] * 4]))
    MX.silu_mul_hip(x, x, out=room[1:].t())
    assert torch.equal(room[1], MX.silu_mul_hip(x, x)[:, 0]) and (room[0].abs() == 2).all()
