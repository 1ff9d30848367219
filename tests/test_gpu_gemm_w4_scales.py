"""Products with 4-bit weights, more closely: beyond 64 rows against weights rounded as they are there, group by group steps and zero points where sums are exact, and the same
rows on both sides of 64."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402
from test_gpu_gemm_w4 import call, problem  # noqa: E402

pytestmark = pytest.mark.gpu
# What f32 sums of K terms of either sign may be off, of the sum of their magnitudes: K / 16 steps that lose 2^-23 of a partial sum each, which stays within 4 sqrt K of a
# term's root mean square, where the magnitudes are 0.6 K of it: 0.4 sqrt K 2^-23, under 2^-17 up to K = 8192.  One k left out is 2^-13 there.
SUMS = 2.0 ** -17


def weights(w, scales, z, group, rounded=None):
    q = torch.stack((w % 16, w // 16), -1).view(w.shape[0], -1).double()
    full = (q - (z.double().repeat_interleave(group, 1) if z is not None else 8.0)) * scales.double().repeat_interleave(group, 1)
    return full if rounded is None else full.to(rounded).double()  # a product of 5 and 11 bits: one rounding


# beyond a cluster's share of K, tiles of 128 and 256 rows, weights made first; K that ends inside a chunk of 128 and of 256
SHAPES = [(65, 264, 512, 64), (100, 2000, 1024, 128), (130, 77, 352, 32), (200, 16400, 256, 32), (300, 1024, 1536, 128), (513, 264, 8192, 32), (641, 4001, 544, 32),
          (130, 16384, 384, 64), (1030, 2056, 512, 128), (1100, 2049, 1024, 64), (1025, 2048, 8192, 32), (96, 300, 160, 32), (70, 130, 4128, 32)]


@pytest.mark.parametrize("m,n,k,group", SHAPES)
@pytest.mark.parametrize("dtype,a_dtype,zeros", [("bf16", "bf16", True), ("f16", "i8", True), ("bf16", "i8", False), ("f16", "f16", False)])
def test_against_rounded_weights(dev, pkg, dtype, a_dtype, zeros, m, n, k, group):
    a, a_scales, w, scales, z = problem(m * 17 + n, dtype, a_dtype, m, n, k, group, zeros)
    c = torch.empty((m, n), dtype=u.TORCH[dtype], device=u.GPU)
    call(pkg, dev, dtype, a_dtype, group, a, a_scales, w, scales, z, c)
    full = weights(w, scales, z, group, u.TORCH[dtype])
    x = a.double() if a_scales is None else a.double() * a_scales.double()[:, None]
    ref, mag = x @ full.T, x.abs() @ full.abs().T
    # C is rounded once
    tol = u.HALF_ULP[dtype] * 1.01 * ref.abs() + SUMS * mag + u.SMALLEST[dtype]
    err = (c.double() - ref).abs()
    assert (err <= tol).all(), (float((err - tol).max()), int((err > tol).sum()))
    assert dev.status() == 0


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype,a_dtype,m,n,k", [("bf16", "bf16", 5, 300, 1024), ("f16", "i8", 40, 300, 1024), ("bf16", "i8", 80, 300, 1152), ("f16", "f16", 150, 16400, 384),
                                                 ("bf16", "bf16", 300, 600, 1408), ("f16", "i8", 300, 600, 1408), ("bf16", "bf16", 1040, 2100, 1024),
                                                 ("f16", "f16", 1040, 2100, 1024), ("bf16", "i8", 1040, 2100, 1024)])
def test_every_group_has_its_own_scale_and_zero_point(dev, pkg, dtype, a_dtype, m, n, k, group):
    """Powers of two and small whole numbers: every sum is exact, C is rounded once."""
    g, t = u.gen(m + n + group), u.TORCH[dtype]
    a = torch.randint(-3, 4, (m, k), generator=g, device=u.GPU)
    w = torch.randint(0, 256, (n, k // 2), generator=g, device=u.GPU, dtype=torch.uint8)
    scales = torch.exp2(torch.randint(-3, 2, (n, k // group), generator=g, device=u.GPU).float()).to(t)
    z = torch.randint(0, 16, (n, k // group), generator=g, device=u.GPU, dtype=torch.uint8)
    steps = torch.exp2(torch.randint(-2, 3, (m,), generator=g, device=u.GPU).float()) if a_dtype == "i8" else None
    a = a.to(torch.int8) if a_dtype == "i8" else a.to(t)
    c = torch.empty((m, n), dtype=t, device=u.GPU)
    call(pkg, dev, dtype, a_dtype, group, a, steps, w, scales, z, c)
    ref = a.double() @ weights(w, scales, z, group).T
    if steps is not None:
        ref = ref * steps.double()[:, None]
    assert torch.equal(c, ref.float().to(t))
    if a_dtype != "i8":
        a[m // 2, k - 7] = float("nan")
        call(pkg, dev, dtype, a_dtype, group, a, steps, w, scales, z, c)
        assert torch.isnan(c[m // 2]).all()
        c[m // 2] = 0
        ref[m // 2] = 0
        assert torch.equal(c, ref.float().to(t))


@pytest.mark.parametrize("dtype,a_dtype", [("bf16", "bf16"), ("f16", "f16"), ("f16", "i8")])
def test_rows_on_both_sides_of_64(dev, pkg, dtype, a_dtype):
    """A row's result differs by its weights' rounding alone."""
    a, a_scales, w, scales, z = problem(9, dtype, a_dtype, 65, 500, 1024, 64, True)
    few, more = (torch.empty((m, 500), dtype=u.TORCH[dtype], device=u.GPU) for m in (64, 65))
    call(pkg, dev, dtype, a_dtype, 64, a[:64], None if a_scales is None else a_scales[:64], w, scales, z, few)
    call(pkg, dev, dtype, a_dtype, 64, a, a_scales, w, scales, z, more)
    x = a.double() if a_scales is None else a.double() * a_scales.double()[:, None]
    exact, rounded = (x[:64] @ weights(w, scales, z, 64, r).T for r in (None, u.TORCH[dtype]))
    mag = x[:64].abs() @ weights(w, scales, z, 64).abs().T
    for c, ref in ((few, exact), (more[:64], rounded)):
        assert ((c.double() - ref).abs() <= u.HALF_ULP[dtype] * 1.01 * ref.abs() + SUMS * mag + u.SMALLEST[dtype]).all()
