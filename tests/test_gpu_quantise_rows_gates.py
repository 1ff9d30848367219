"""silu(gate) * up value by value: rows of one column, whose step alone tells the value (127 times it, in magnitude), so that small values are not judged beside a row's largest one."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu


def steps(pkg, dev, dtype, gate, up):
    """The steps of rows of `gate.shape[1]` equal columns, all of the same value."""
    rows, cols = gate.shape
    y, scales = torch.zeros((rows, cols), dtype=torch.int8, device=u.GPU), torch.zeros(rows, device=u.GPU)
    dev.quantise_rows(u.codes(pkg.capi)[dtype], rows, cols, u.ptr(gate), u.ptr(y), u.ptr(scales), up=u.ptr(up), stream=u.stream())
    return y, scales


def bound(gate):
    """How far f32 may be, relative: x * log2(e) rounded, with a rounded constant (2^-24 and 2^-26.1 of |x| in the exponential, which counts as exp(-x) / (1 + exp(-x))); the exponential 2^-22,
    the sum 2^-24, the reciprocal 2^-23 and, where it is below 2^-126, another 2^-22 (21 bits are left at 2^-128); two products 2^-24 each; the step's constant and product 2^-24 each."""
    e = torch.exp(-gate)
    weight = torch.where(torch.isinf(e), torch.ones_like(e), e / (1 + e))
    return weight * gate.abs() * 2.0 ** -24 * 1.24 + 2.0 ** -22 + 2.0 ** -24 + 2.0 ** -23 + 2.0 ** -22 + 4 * 2.0 ** -24


# one column: the kernel for rows that start anywhere; four and eight: vectors of f32, and of 16 bits; 9000 and 33000: rows in registers of a CTA, and read twice
@pytest.mark.parametrize("dtype,cols,step", [("f32", 1, 0.013), ("f32", 4, 0.013), ("f32", 9000, 7.1), ("f32", 33000, 19.0), ("bf16", 8, 0.07), ("f16", 8, 0.07), ("f16", 1, 0.07)])
@pytest.mark.parametrize("scale", [1.0, -1.0, 2.0 ** 100])
def test_each_value(dev, pkg, dtype, cols, step, scale):
    """From where exp(-x) is finite up to where it is nothing beside 1, among them the gates whose reciprocal is below the smallest normal f32."""
    if dtype == "f16" and scale > 1:
        scale = 2.0 ** 15
    t = u.TORCH[dtype]
    low = -88.7
    x = torch.cat((torch.arange(low, 60.0, step, dtype=torch.float64), torch.arange(low, -87.2, 0.01, dtype=torch.float64) if cols < 100 else torch.tensor([-88.0, -87.5], dtype=torch.float64)))
    x = x.to(t).to(u.GPU)
    x = x[(x != 0) & (x.double() >= -88.72)]
    gate = x[:, None].expand(-1, cols).contiguous()
    up = torch.full_like(gate, scale)
    y, scales = steps(pkg, dev, dtype, gate, up)
    g = x.double()
    want = (g / (1 + torch.exp(-g)) * scale).abs()
    keep = want < 2.0 ** 127
    off = ((scales.double() * 127 - want).abs() / want)[keep]
    # a step below 2^-126 is rounded to a multiple of 2^-149; 1/127 of a value of 2^-121.5 is that small
    assert (off <= bound(g)[keep] + (127 * 2.0 ** -149 / want)[keep]).all(), float((off / bound(g)[keep]).max())
    assert (scales > 0).all()
    # the number beside the step: 127, or 126 where a step among the smallest numbers was rounded up
    assert ((y.double() * scales.double()[:, None]).abs() - want[:, None]).abs()[keep].le((0.5 * scales.double() + want * bound(g))[keep][:, None] + 127 * 2.0 ** -149).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gates_whose_exponential_overflows_count_as_zero(dev, pkg, dtype):
    x = torch.tensor([-88.75, -89.0, -100.0, -1000.0, -3e38], device=u.GPU).to(u.TORCH[dtype])[:, None]
    y, scales = steps(pkg, dev, dtype, x.contiguous(), torch.full_like(x, 2.0 ** 100))
    assert (y == 0).all() and (scales == 0).all()
