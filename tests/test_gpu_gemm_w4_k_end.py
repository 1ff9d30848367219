"""Products with 4-bit weights whose K ends inside a chunk of 128: what lies behind it has no weight, whatever its scale would make of it."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402
from test_gpu_gemm_w4 import call  # noqa: E402

pytestmark = pytest.mark.gpu
# What f32 sums of K terms of either sign may be off, of the sum of their magnitudes: K / 16 steps that lose 2^-23 of a partial sum each, which stays within 4 sqrt K of a
# term's root mean square, where the magnitudes are 0.6 K of it: 0.4 sqrt K 2^-23, under 2^-17 up to K = 8192.  One k left out is 2^-13 there.
SUMS = 2.0 ** -17


def weights(w, scales, z, group, rounded=None):
    q = torch.stack((w % 16, w // 16), -1).view(w.shape[0], -1).double()
    full = (q - (z.double().repeat_interleave(group, 1) if z is not None else 8.0)) * scales.double().repeat_interleave(group, 1)
    return full if rounded is None else full.to(rounded).double()  # a product of 5 and 11 bits: one rounding


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k", [(66, 200, 160), (300, 16400, 96), (80, 256, 288), (40, 256, 288)])
def test_large_scales(dev, pkg, m, n, k, zeros):
    """f16, (q - zero) * scale of the last group within f16, 8 or its zero point times that scale beyond it."""
    g = u.gen(m + k)
    a = (u.normal(g, (m, k)) * 2.0 ** -10).half()
    w = torch.randint(0, 256, (n, k // 2), generator=g, device=u.GPU, dtype=torch.uint8)
    scales = torch.full((n, k // 32), 1.0, dtype=torch.float16, device=u.GPU)
    scales[:, -1] = 9000.0
    z = torch.full((n, k // 32), 15, dtype=torch.uint8, device=u.GPU) if zeros else None
    nibbles = torch.randint(9, 15, (n, 32), generator=g, device=u.GPU, dtype=torch.uint8) if zeros else torch.randint(5, 12, (n, 32), generator=g, device=u.GPU, dtype=torch.uint8)
    w[:, -16:] = nibbles[:, 0::2] | (nibbles[:, 1::2] << 4)  # at most six or three steps from the zero point
    full = weights(w, scales, z, 32)
    assert full.abs().max() <= 65504
    c = torch.empty((m, n), dtype=torch.float16, device=u.GPU)
    call(pkg, dev, "f16", "f16", 32, a, None, w, scales, z, c)
    rounded = full.half().double() if m > 64 else full
    ref, mag = a.double() @ rounded.T, a.double().abs() @ rounded.abs().T
    assert torch.isfinite(c).all()
    assert ((c.double() - ref).abs() <= u.HALF_ULP["f16"] * 1.01 * ref.abs() + SUMS * mag + u.SMALLEST["f16"]).all()
