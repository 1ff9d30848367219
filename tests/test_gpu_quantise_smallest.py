"""Rows in 8 bits whose largest magnitude is among the smallest f32 numbers, where a step is a few times 2^-149: x / step would be up to 190 over the nearest one, or the step 0."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu
TOPS = [1, 2, 63, 64, 127, 128, 150, 190, 191, 254, 255, 256, 381, 382, 383, 1000, 30000, 190000, 8388607]


@pytest.mark.parametrize("cols", [40, 1001, 4096, 9001])  # a warp a row on vectors; rows that start anywhere, short and long
def test_numbers_keep_their_sign_and_range(dev, pkg, cols):
    ramp = torch.linspace(-1, 1, cols, dtype=torch.float64)
    units = torch.stack([torch.round(ramp * top) for top in TOPS])  # of 2^-149
    units[:, 0] = -torch.tensor(TOPS).double()
    bits = units.abs().to(torch.int32) | (units < 0).to(torch.int32) << 31
    x = bits.view(torch.float32).to(u.GPU)
    y, scales = torch.empty(x.shape, dtype=torch.int8, device=u.GPU), torch.empty(len(TOPS), device=u.GPU)
    dev.add_rms_norm(pkg.capi.F32, len(TOPS), cols, 1.0, u.ptr(x), 0, 0, 0, u.ptr(y), out_dtype=pkg.capi.I8, scales=u.ptr(scales), stream=u.stream())
    # the squares are 0 and eps is 1: scales are the steps
    steps = scales.cpu().view(torch.int32).double()[:, None]
    exact = torch.tensor(TOPS).double()[:, None] / 127
    assert (steps >= 1).all() and ((steps - exact).abs() <= 1).all()
    q = y.cpu().double()
    assert torch.equal(q, torch.round(units / steps)) and q.abs().max() == 127
    assert dev.status() == 0
