"""The norm that adds the residual: against the definition in 64 bits, rows and widths where vectors end, 8-bit rows number by number."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-5
# one row, a few, many; widths of one element, below a vector, odd, of whole vectors, and longer than a CTA keeps in registers
SHAPES = [(1, 4096), (3, 1), (5, 7), (2, 130), (7, 1000), (300, 257), (1200, 512), (33, 5001), (4, 16384), (2, 40000), (3, 33001), (2, 100001)]


def call(pkg, dev, dtype, out, x, res, w, total, y, scales=None, eps=EPS):
    c = u.codes(pkg.capi)
    dev.add_rms_norm(c[dtype], x.shape[0], x.shape[1], eps, u.ptr(x), u.ptr(res), u.ptr(total), u.ptr(w), u.ptr(y), out_dtype=c[out], scales=u.ptr(scales),
                     stream=u.stream())


def close(got, want, dtype, what):
    # one rounding of a value that f32 arithmetic gives to 2e-6 (sums of squares in a tree: log2(cols) + cols / threads roundings of positive terms, halved by
    # the root)
    tol = (u.HALF_ULP[dtype] + 4e-6) * want.abs() + u.SMALLEST[dtype]
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), (got.double() - want).abs().max())


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_storage_type(dev, pkg, dtype, rows, cols):
    g, t = u.gen(rows * 7 + cols), u.TORCH[dtype]
    x, res, w = u.normal(g, (rows, cols)).to(t), u.normal(g, (rows, cols), 3.0).to(t), (1 + u.normal(g, (cols,), 0.3)).to(t)
    for with_res, with_w, with_sum in ((True, True, True), (False, False, False), (True, False, False), (False, True, True)):
        y, total = torch.full_like(x, 7), torch.full_like(x, 7) if with_sum else None
        call(pkg, dev, dtype, dtype, x, res if with_res else None, w if with_w else None, total, y)
        h = x.double() + (res.double() if with_res else 0)
        want = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * (w.double() if with_w else 1)
        close(y, want, dtype, (with_res, with_w))
        if with_sum:
            assert torch.equal(total, h.float().to(t))  # h in f32 is one rounding, exact for 16-bit terms unless they are far apart
    assert dev.status() == 0


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_eight_bits(dev, pkg, dtype, rows, cols):
    g, t = u.gen(rows * 5 + cols), u.TORCH[dtype]
    x, res, w = u.normal(g, (rows, cols)).to(t), u.normal(g, (rows, cols), 3.0).to(t), (1 + u.normal(g, (cols,), 0.3)).to(t)
    if rows > 1:
        x[1] = 0
        res[1] = 0  # a row of zeros: step 0
    y, scales, total = torch.full((rows, cols), 99, dtype=torch.int8, device=u.GPU), torch.full((rows,), 7.0, device=u.GPU), torch.empty_like(x)
    call(pkg, dev, dtype, "i8", x, res, w, total, y, scales)
    h = x.float() + res.float()
    q, step = u.quantise(h * w.float())
    assert torch.equal(y, q)
    want = step.double() * torch.rsqrt(h.double().square().mean(-1) + EPS)
    assert ((scales.double() - want).abs() <= 4e-6 * want).all()
    assert torch.equal(total, h.to(t))


@pytest.mark.parametrize("cols", [512, 1001, 20000])
def test_in_place(dev, pkg, cols):
    """sum over x or over the residual, y over the other."""
    g = u.gen(cols)
    x, res = u.normal(g, (6, cols)).bfloat16(), u.normal(g, (6, cols)).bfloat16()
    h = x.double() + res.double()
    want = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    for over in range(3):
        a, b = x.clone(), res.clone()
        total, y = ((a, b), (b, a), (b, torch.empty_like(a)))[over]
        call(pkg, dev, "bf16", "bf16", a, b, None, total, y)
        close(y, want, "bf16", over)
        assert torch.equal(total, h.float().bfloat16())


@pytest.mark.parametrize("shift", [1, 3, 8])
def test_rows_that_start_anywhere(dev, pkg, shift):
    """Every buffer some elements behind a vector's boundary, none alike."""
    g, rows, cols = u.gen(shift), 5, 776
    flat = [torch.empty(rows * cols + 40, dtype=torch.float16, device=u.GPU) for _ in range(5)]
    x, res, w, total, y = (f[shift * (i + 1) % 11:][:(cols if i == 2 else rows * cols)].view(-1 if i == 2 else rows, cols) for i, f in enumerate(flat))
    x.copy_(u.normal(g, (rows, cols)))
    res.copy_(u.normal(g, (rows, cols)))
    w.copy_(1 + u.normal(g, (1, cols), 0.1))
    call(pkg, dev, "f16", "f16", x, res, w, total, y)
    h = x.double() + res.double()
    close(y, h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w.double(), "f16", shift)
    raw = torch.full((rows * cols + 40,), 55, dtype=torch.int8, device=u.GPU)
    q, scales = raw[shift:][:rows * cols].view(rows, cols), torch.empty(rows, device=u.GPU)
    call(pkg, dev, "f16", "i8", x, res, w, total, q, scales)
    assert torch.equal(q, u.quantise((x.float() + res.float()) * w.float())[0])
    assert (raw[:shift] == 55).all() and (raw[shift + rows * cols:] == 55).all()


def test_what_is_not_finite_stays_in_its_row(dev, pkg):
    x = torch.ones((4, 300), device=u.GPU)
    x[1, 7], x[2, 9] = float("nan"), float("inf")
    y, q, scales = torch.empty_like(x), torch.empty((4, 300), dtype=torch.int8, device=u.GPU), torch.empty(4, device=u.GPU)
    call(pkg, dev, "f32", "f32", x, None, None, None, y)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 9]) and torch.isfinite(y[[0, 3]]).all()
    call(pkg, dev, "f32", "i8", x, None, None, None, q, scales)
    assert torch.isnan(scales[[1, 2]]).all() and torch.isfinite(scales[[0, 3]]).all() and (q[[0, 3]] == 127).all()


def test_refusals(dev, pkg):
    capi, hal = pkg.capi, pkg.hal
    x = torch.zeros(64, device=u.GPU)
    p = x.data_ptr()

    def bad(match, dtype=capi.F32, out=None, rows=2, cols=8, x=p, res=0, total=0, w=0, y=p + 128, scales=0):
        with pytest.raises(hal.KernelError, match=match):
            dev.add_rms_norm(dtype, rows, cols, EPS, x, res, total, w, y, out_dtype=out, scales=scales, stream=u.stream())

    bad("unknown dtype", dtype=7)
    bad("unknown dtype", dtype=capi.I8)
    bad("out_dtype", out=capi.BF16)
    bad("bad shape", rows=-1)
    bad("bad shape", cols=1 << 31)
    bad("null buffer", x=0)
    bad("null buffer", y=0)
    bad("needs scales", out=capi.I8)
    bad("same buffer", total=p + 128)
    bad("cannot be x", out=capi.I8, y=p, scales=p + 200)
    bad("element boundary", x=p + 2)
    dev.add_rms_norm(capi.F32, 0, 8, EPS, 0, 0, 0, 0, 0, stream=u.stream())  # nothing to do
    dev.add_rms_norm(capi.F32, 8, 0, EPS, 0, 0, 0, 0, 0, stream=u.stream())
