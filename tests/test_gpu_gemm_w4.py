"""Products with 4-bit weights against the definition in 64 bits: rows from one to a prompt's, odd numbers of outputs, every group size, zero points."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu


def problem(seed, dtype, a_dtype, m, n, k, group, zeros):
    g, t = u.gen(seed), u.TORCH[dtype]
    x = u.normal(g, (m, k))
    a, a_scales = u.quantise(x) if a_dtype == "i8" else (x.to(t), None)
    w = torch.randint(0, 256, (n, k // 2), generator=g, device=u.GPU, dtype=torch.uint8)
    scales = (torch.exp(u.normal(g, (n, k // group), 0.5)) * 0.05).to(t)
    z = torch.randint(0, 16, (n, k // group), generator=g, device=u.GPU, dtype=torch.uint8) if zeros else None
    return a, a_scales, w, scales, z


def reference(a, a_scales, w, scales, z, group):
    """C and the sum of the terms' magnitudes."""
    q = torch.stack((w % 16, w // 16), -1).view(w.shape[0], -1).double()
    full = (q - (z.double().repeat_interleave(group, 1) if z is not None else 8.0)) * scales.double().repeat_interleave(group, 1)
    a = a.double() if a_scales is None else a.double() * a_scales.double()[:, None]
    return a @ full.T, a.abs() @ full.abs().T


def call(pkg, dev, dtype, a_dtype, group, a, a_scales, w, scales, z, c):
    k = u.codes(pkg.capi)
    dev.gemm_w4(k[dtype], c.shape[0], c.shape[1], a.shape[1], group, u.ptr(a), u.ptr(w), u.ptr(scales), u.ptr(c), a_dtype=k[a_dtype], a_scales=u.ptr(a_scales),
                w_zeros=u.ptr(z), stream=u.stream())


def check(got, ref, mag, dtype, m):
    # C rounded once; f32 sums of K terms lose at most 2^-23 of the magnitudes a step of 16, 2^-16 in all up to K = 2048, and random signs keep far below;
    # more than 64 rows: each weight rounded once more
    tol = u.HALF_ULP[dtype] * 1.01 * ref.abs() + (2.0 ** -16 + (u.HALF_ULP[dtype] if m > 64 else 0)) * mag + u.SMALLEST[dtype]
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float(err.max()))


SHAPES = [(1, 1, 32, 32), (1, 64, 128, 128), (1, 4096, 4096, 128), (2, 1000, 1024, 64), (3, 17, 96, 32), (4, 130, 2048, 128), (7, 513, 320, 64), (8, 256, 512, 32),
          (9, 333, 1152, 128), (13, 31, 4096, 64), (16, 2048, 1024, 128), (17, 100, 256, 128), (31, 4099, 640, 32), (32, 512, 2048, 64), (33, 129, 1280, 128),
          (48, 640, 384, 128), (64, 1000, 2048, 32), (65, 264, 512, 64), (100, 2000, 1024, 128), (130, 77, 352, 32), (300, 1024, 1536, 128), (513, 520, 256, 64),
          (1, 20000, 256, 128), (5, 48, 16384, 128), (70, 8, 64, 64)]


@pytest.mark.parametrize("m,n,k,group", SHAPES)
@pytest.mark.parametrize("dtype,a_dtype,zeros", [("bf16", "bf16", False), ("f16", "i8", True), ("bf16", "i8", False), ("f16", "f16", True)])
def test_against_the_definition(dev, pkg, dtype, a_dtype, zeros, m, n, k, group):
    a, a_scales, w, scales, z = problem(m * 31 + n, dtype, a_dtype, m, n, k, group, zeros)
    raw = torch.full((m * n + 16,), 77.0, dtype=u.TORCH[dtype], device=u.GPU)
    c = raw[:m * n].view(m, n)
    for _ in range(2):
        call(pkg, dev, dtype, a_dtype, group, a, a_scales, w, scales, z, c)
    ref, mag = reference(a, a_scales, w, scales, z, group)
    check(c, ref, mag, dtype, m)
    assert (raw[m * n:] == 77).all()
    assert dev.status() == 0


@pytest.mark.parametrize("m", [1, 12, 80])
def test_a_result_that_starts_anywhere(dev, pkg, m):
    """C, scales and zero points one element behind a vector's boundary."""
    a, a_scales, w, scales, z = problem(m, "bf16", "bf16", m, 200, 256, 64, True)
    raw, s1 = torch.zeros(m * 200 + 1, dtype=torch.bfloat16, device=u.GPU), torch.zeros(scales.numel() + 1, dtype=torch.bfloat16, device=u.GPU)
    z1 = torch.zeros(z.numel() + 1, dtype=torch.uint8, device=u.GPU)
    s1[1:], z1[1:] = scales.view(-1), z.view(-1)
    c = raw[1:].view(m, 200)
    call(pkg, dev, "bf16", "bf16", 64, a, a_scales, w, s1[1:], z1[1:], c)
    ref, mag = reference(a, a_scales, w, scales, z, 64)
    check(c, ref, mag, "bf16", m)


@pytest.mark.parametrize("m", [1, 20, 100])
def test_exact_where_sums_are(dev, pkg, m):
    """Whole numbers with steps that are powers of two come out bit for bit: one rounding."""
    g = u.gen(m)
    a = torch.randint(-3, 4, (m, 512), generator=g, device=u.GPU).bfloat16()
    w = torch.randint(0, 256, (192, 256), generator=g, device=u.GPU, dtype=torch.uint8)
    scales = torch.full((192, 4), 0.5, dtype=torch.bfloat16, device=u.GPU)
    c = torch.empty((m, 192), dtype=torch.bfloat16, device=u.GPU)
    call(pkg, dev, "bf16", "bf16", 128, a, None, w, scales, None, c)
    assert torch.equal(c, reference(a, None, w, scales, None, 128)[0].bfloat16())


@pytest.mark.parametrize("m", [2, 30, 90])
def test_what_is_not_finite_stays_in_its_row(dev, pkg, m):
    a, _, w, scales, _ = problem(m, "f16", "f16", m, 256, 512, 128, False)
    a[1, 100] = float("nan")
    c = torch.empty((m, 256), dtype=torch.float16, device=u.GPU)
    call(pkg, dev, "f16", "f16", 128, a, None, w, scales, None, c)
    assert torch.isnan(c[1]).all() and torch.isfinite(c[0]).all() and torch.isfinite(c[2:]).all()


@pytest.mark.parametrize("m,n,k,group", [(513, 264, 8192, 32), (520, 2049, 1024, 64), (641, 4001, 544, 32), (300, 8200, 512, 128), (385, 4801, 640, 64), (1030, 1028, 2048, 128)])
@pytest.mark.parametrize("dtype,a_dtype,zeros", [("bf16", "bf16", True), ("f16", "i8", True), ("bf16", "i8", False), ("f16", "f16", False)])
def test_rows_enough_to_make_the_weights_first(dev, pkg, dtype, a_dtype, zeros, m, n, k, group):
    a, a_scales, w, scales, z = problem(m + n, dtype, a_dtype, m, n, k, group, zeros)
    raw = torch.full((m * n + 16,), 77.0, dtype=u.TORCH[dtype], device=u.GPU)
    ref, mag = reference(a, a_scales, w, scales, z, group)
    for start in (0, 1):  # C on a vector's boundary and off it
        c = raw[start:start + m * n].view(m, n)
        call(pkg, dev, dtype, a_dtype, group, a, a_scales, w, scales, z, c)
        check(c, ref, mag, dtype, m)
        assert (raw[m * n + start:] == 77).all()
    assert dev.status() == 0


@pytest.mark.parametrize("m,n,k,group", [(200, 16400, 256, 32), (130, 16384, 384, 64), (1030, 2056, 512, 128), (1100, 2049, 1024, 64), (1025, 2048, 544, 32)])
@pytest.mark.parametrize("dtype,a_dtype,zeros", [("bf16", "bf16", True), ("f16", "i8", True), ("bf16", "i8", False), ("f16", "f16", False)])
def test_many_tiles_and_many_rows(dev, pkg, dtype, a_dtype, zeros, m, n, k, group):
    """Tiles of 256 rows; weights made 16-bit ones first."""
    test_rows_enough_to_make_the_weights_first(dev, pkg, dtype, a_dtype, zeros, m, n, k, group)


def test_many_rows_exact_and_not_finite(dev, pkg):
    g = u.gen(6)
    a = torch.randint(-3, 4, (1040, 1024), generator=g, device=u.GPU).half()
    w = torch.randint(0, 256, (2100, 512), generator=g, device=u.GPU, dtype=torch.uint8)
    scales = torch.full((2100, 8), 0.5, dtype=torch.float16, device=u.GPU)
    c = torch.empty((1040, 2100), dtype=torch.float16, device=u.GPU)
    ref = reference(a, None, w, scales, None, 128)[0].half()
    call(pkg, dev, "f16", "f16", 128, a, None, w, scales, None, c)
    assert torch.equal(c, ref)
    a[129, 7] = float("nan")
    call(pkg, dev, "f16", "f16", 128, a, None, w, scales, None, c)
    assert torch.isnan(c[129]).all()
    c[129] = ref[129]
    assert torch.equal(c, ref)


def test_rows_enough_to_make_the_weights_first_exact_and_not_finite(dev, pkg):
    g = u.gen(5)
    a = torch.randint(-3, 4, (530, 1024), generator=g, device=u.GPU).bfloat16()
    w = torch.randint(0, 256, (2100, 512), generator=g, device=u.GPU, dtype=torch.uint8)
    scales = torch.full((2100, 8), 0.5, dtype=torch.bfloat16, device=u.GPU)
    c = torch.empty((530, 2100), dtype=torch.bfloat16, device=u.GPU)
    call(pkg, dev, "bf16", "bf16", 128, a, None, w, scales, None, c)
    ref = reference(a, None, w, scales, None, 128)[0].bfloat16()
    assert torch.equal(c, ref)
    a[129, 7] = float("nan")
    call(pkg, dev, "bf16", "bf16", 128, a, None, w, scales, None, c)
    assert torch.isnan(c[129]).all()
    c[129] = ref[129]
    assert torch.equal(c, ref)


def test_no_terms(dev, pkg):
    capi = pkg.capi
    c = torch.full((3, 5), 9.0, dtype=torch.bfloat16, device=u.GPU)
    dev.gemm_w4(capi.BF16, 3, 5, 0, 128, 0, 0, 0, u.ptr(c), stream=u.stream())
    assert (c == 0).all()


def test_refusals(dev, pkg):
    capi, hal = pkg.capi, pkg.hal
    x = torch.zeros(4096, device=u.GPU)
    p = x.data_ptr()

    def bad(match, dtype=capi.BF16, m=2, n=8, k=128, group=128, a=p, w=p, s=p, c=p + 8192, a_dtype=None, a_scales=0):
        with pytest.raises(hal.KernelError, match=match):
            dev.gemm_w4(dtype, m, n, k, group, a, w, s, c, a_dtype=a_dtype, a_scales=a_scales, stream=u.stream())

    bad("dtype must be", dtype=capi.F32)
    bad("a_dtype", a_dtype=capi.F16)
    bad("group must be", group=96)
    bad("bad shape", m=-1)
    bad("bad shape", k=1 << 31)
    bad("multiple of group", k=160)
    bad("null buffer", a=0)
    bad("null buffer", w=0)
    bad("null buffer", s=0)
    bad("null buffer", c=0)
    bad("a_scales", a_dtype=capi.I8)
    bad("16-byte aligned", a=p + 2)
    bad("16-byte aligned", w=p + 4)
    bad("element boundary", c=p + 1)
    dev.gemm_w4(capi.BF16, 0, 8, 128, 128, 0, 0, 0, 0, stream=u.stream())  # nothing to do
