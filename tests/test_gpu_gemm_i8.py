"""Products in 8 bits against the definition in 64 bits: one row to a prompt's, odd numbers of everything, pitches, buffers that start anywhere."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu


def problem(seed, m, n, k):
    g = u.gen(seed)
    a = torch.randint(-128, 128, (m, k), generator=g, device=u.GPU, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, device=u.GPU, dtype=torch.int8)
    return a, torch.exp(u.normal(g, (m,))) * 0.01, w, torch.exp(u.normal(g, (n,))) * 0.01


def reference(a, a_scales, w, w_scales):
    """The sums in f64 are exact (below 2^53), so C is off by the roundings of two products."""
    return (a.double() @ w.double().T) * a_scales.double()[:, None] * w_scales.double()


def call(pkg, dev, dtype, a, a_scales, w, w_scales, c, lda=0, ldw=0, ldc=0, shape=None):
    m, n, k = shape or (c.shape[0], c.shape[1], a.shape[1])
    dev.gemm_i8(u.codes(pkg.capi)[dtype], m, n, k, u.ptr(a), u.ptr(a_scales), u.ptr(w), u.ptr(w_scales), u.ptr(c), lda=lda, ldw=ldw, ldc=ldc, stream=u.stream())


def check(got, ref, dtype):
    # the sum rounded to f32, two f32 products, one rounding to dtype: 2^-24 three times (1 + 2^-20 for their products), and dtype's half step
    tol = (3.001 * 2.0 ** -24 + (0 if dtype == "f32" else 1.001 * u.HALF_ULP[dtype])) * ref.abs() + u.SMALLEST[dtype]
    err = (got.double() - ref).abs()
    finite = ref.abs() < (65504 if dtype == "f16" else 3e38)
    assert (err[finite] <= tol[finite]).all(), (float((err - tol)[finite].max()), float(err[finite].max()))


SHAPES = [(1, 1, 16), (1, 1, 1), (1, 64, 128), (1, 4096, 4096), (2, 1000, 1024), (3, 17, 96), (4, 130, 2048), (7, 513, 320), (9, 333, 1152), (16, 2048, 1024), (17, 100, 256),
          (31, 4099, 640), (33, 129, 1280), (48, 640, 384), (64, 1000, 2048), (65, 264, 512), (100, 2000, 1024), (129, 77, 352), (130, 257, 4112), (300, 1024, 1536), (513, 520, 256),
          (777, 1003, 272), (1, 20000, 256), (5, 48, 16384), (70, 8, 64), (2, 40, 131056), (1000, 3000, 128), (2100, 2100, 64), (257, 2049, 8192), (4097, 640, 1040)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_against_the_definition(dev, pkg, dtype, m, n, k):
    a, a_scales, w, w_scales = problem(m * 31 + n, m, n, k)
    raw = torch.full((m * n + 16,), 77.0, dtype=u.TORCH[dtype], device=u.GPU)
    c = raw[:m * n].view(m, n)
    for _ in range(2):
        call(pkg, dev, dtype, a, a_scales, w, w_scales, c)
    check(c, reference(a, a_scales, w, w_scales), dtype)
    assert (raw[m * n:] == 77).all()
    assert dev.status() == 0


@pytest.mark.parametrize("m,n,k", [(1, 33, 17), (5, 100, 999), (40, 257, 63), (200, 300, 1001), (600, 1100, 4095), (3, 5, 131071)])
def test_rows_that_start_anywhere(dev, pkg, m, n, k):
    """K is no multiple of 16: both operands are copied."""
    a, a_scales, w, w_scales = problem(k, m, n, k)
    c = torch.empty((m, n), dtype=torch.float32, device=u.GPU)
    call(pkg, dev, "f32", a, a_scales, w, w_scales, c)
    check(c, reference(a, a_scales, w, w_scales), "f32")


@pytest.mark.parametrize("m,n,k,lda,ldw,ldc,off", [(9, 130, 100, 112, 128, 131, 0), (9, 130, 100, 101, 128, 131, 0), (9, 130, 96, 96, 99, 136, 0), (20, 64, 64, 0, 0, 0, 1),
                                                   (300, 513, 320, 337, 352, 520, 3), (600, 1024, 512, 512, 512, 1032, 16), (1100, 1024, 512, 528, 544, 2000, 0)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_pitches_and_offsets(dev, pkg, dtype, m, n, k, lda, ldw, ldc, off):
    """Rows apart, buffers off vectors' boundaries; nothing but the result is written."""
    g = u.gen(m)
    la, lw, lc = lda or k, ldw or k, ldc or n
    raw_a = torch.randint(-128, 128, (m * la + off,), generator=g, device=u.GPU, dtype=torch.int8)
    raw_w = torch.randint(-128, 128, (n * lw + off,), generator=g, device=u.GPU, dtype=torch.int8)
    raw_c = torch.full((m * lc + off,), 5.0, dtype=u.TORCH[dtype], device=u.GPU)
    a, w, c = raw_a[off:].view(m, la), raw_w[off:].view(n, lw), raw_c[off:].view(m, lc)
    a_scales, w_scales = torch.exp(u.normal(g, (m,))), torch.exp(u.normal(g, (n,)))
    call(pkg, dev, dtype, a, a_scales, w, w_scales, c, lda, ldw, ldc, (m, n, k))
    check(c[:, :n], reference(a[:, :k], a_scales, w[:, :k], w_scales), dtype)
    assert (c[:, n:] == 5).all() and (raw_c[:off] == 5).all()


@pytest.mark.parametrize("m", [1, 20, 100, 700])
def test_sums_are_exact(dev, pkg, m):
    """With steps of one an f32 result is the sum, where f32 has it: the largest of both signs among them."""
    k = 1040
    a, _, w, _ = problem(m, m, 300, k)
    a[0], w[0], w[1] = -128, -128, 127
    one = torch.ones(1000, device=u.GPU)
    c = torch.empty((m, 300), dtype=torch.float32, device=u.GPU)
    call(pkg, dev, "f32", a, one[:m], w, one[:300], c)
    assert torch.equal(c.double(), (a.double() @ w.double().T).float().double())
    assert float(c[0, 0]) == 128 * 128 * k and float(c[0, 1]) == -128 * 127 * k


def test_the_longest_sum(dev, pkg):
    k = 131071
    a, w = torch.full((2, k), -128, dtype=torch.int8, device=u.GPU), torch.full((3, k), -128, dtype=torch.int8, device=u.GPU)
    w[1] = 127
    one = torch.ones(3, device=u.GPU)
    c = torch.empty((2, 3), dtype=torch.float32, device=u.GPU)
    call(pkg, dev, "f32", a, one, w, one, c)
    assert c[:, 0].tolist() == [float(torch.tensor(16384 * k, dtype=torch.float64).float())] * 2
    assert c[:, 1].tolist() == [float(torch.tensor(-128 * 127 * k, dtype=torch.float64).float())] * 2


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (40, 300, 256), (600, 1500, 512)])
def test_rows_that_are_not_finite(dev, pkg, m, n, k):
    """A step of NaN, of a row of a or of w, is NaN in its row or column of C and nowhere else."""
    a, a_scales, w, w_scales = problem(1, m, n, k)
    a_scales[m // 2], w_scales[n // 3] = float("nan"), float("nan")
    c = torch.empty((m, n), dtype=torch.bfloat16, device=u.GPU)
    call(pkg, dev, "bf16", a, a_scales, w, w_scales, c)
    bad = torch.zeros((m, n), dtype=torch.bool, device=u.GPU)
    bad[m // 2], bad[:, n // 3] = True, True
    assert torch.equal(torch.isnan(c), bad)


def test_nothing_to_sum(dev, pkg):
    c = torch.full((3, 10), 4.0, dtype=torch.bfloat16, device=u.GPU)
    dev.gemm_i8(pkg.capi.BF16, 3, 7, 0, 0, 0, 0, 0, u.ptr(c), ldc=10, stream=u.stream())
    assert (c[:, :7] == 0).all() and (c[:, 7:] == 4).all()
    dev.gemm_i8(pkg.capi.BF16, 0, 7, 16, 0, 0, 0, 0, 0, stream=u.stream())


@pytest.mark.parametrize("m", [4, 700])
def test_captured_on_another_stream_and_replayed(dev, pkg, m):
    """Two graphs of calls that take scratch, replayed in turn with other inputs."""
    n, k = 1100, 501
    side = torch.cuda.Stream()
    a, a_scales, w, w_scales = problem(3, m, n, k)
    out = [torch.empty((m, n), dtype=torch.bfloat16, device=u.GPU) for _ in range(2)]
    call(pkg, dev, "bf16", a, a_scales, w, w_scales, out[0])
    torch.cuda.synchronize()
    graphs = []
    for c in out:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(pkg, dev, "bf16", a, a_scales, w, w_scales, c)
        graphs.append(graph)
    for seed in (5, 6):
        for t, x in zip((a, a_scales, w, w_scales), problem(seed, m, n, k)):
            t.copy_(x)
        for c in out:
            c.zero_()
        for graph in graphs * 2:
            graph.replay()
        for c in out:
            check(c, reference(a, a_scales, w, w_scales), "bf16")
    torch.cuda.synchronize()
    assert dev.status() == 0
