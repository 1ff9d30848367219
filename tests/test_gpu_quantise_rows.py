"""Rows as 8-bit whole numbers and steps, of a tensor and of silu(gate) * up, against the definition: widths from one on, pitches, rows off boundaries, rows that are not
finite."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu


def call(pkg, dev, dtype, x, up, rows, cols, pitch=0, y=None, scales=None):
    y = torch.full((rows * cols + 16,), 99, dtype=torch.int8, device=u.GPU) if y is None else y
    scales = torch.full((rows + 1,), 3.0, device=u.GPU) if scales is None else scales
    dev.quantise_rows(u.codes(pkg.capi)[dtype], rows, cols, u.ptr(x), u.ptr(y), u.ptr(scales), up=u.ptr(up), pitch=pitch, stream=u.stream())
    return y, scales


def check(y, scales, v, slack):
    """v in f64; `slack`: how far f32 may be from it, relative to a value."""
    top = v.abs().amax(-1)
    step = top / 127
    assert ((scales.double() - step).abs() <= (slack + 2.0 ** -23) * step + 2.0 ** -149).all()
    # whole numbers: half a step from the value, and what f32 loses of a value and its quotient (127 of them at most)
    err = (y.double() * scales.double()[:, None] - v).abs()
    assert (err <= scales.double()[:, None] * 0.5 + (slack + 2.0 ** -22) * top[:, None] + 2.0 ** -149).all()
    assert (y.abs().amax(-1)[top > 0] == 127).all() and (y[top == 0] == 0).all() and (scales[top == 0] == 0).all()


WIDTHS = [1, 2, 7, 8, 31, 64, 100, 255, 256, 513, 520, 1024, 1025, 2048, 4096, 4099, 5000, 8192, 8200, 14336, 16384, 28672, 32776, 40001]


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_by_the_definitions_own_operations(dev, pkg, dtype, cols):
    """Without a gate the whole numbers and steps are those of the definition in f32, bit for bit."""
    rows = 1 if cols > 30000 else 9 if cols > 2000 else 37
    x = (u.normal(u.gen(cols), (rows, cols)) * torch.exp(u.normal(u.gen(1), (rows, 1), 2.0))).to(u.TORCH[dtype])
    if rows > 5:
        x[5] = 0
    for _ in range(2):
        y, scales = call(pkg, dev, dtype, x, None, rows, cols)
    q, step = u.quantise(x.float())
    assert torch.equal(y[:rows * cols].view(rows, cols), q) and torch.equal(scales[:rows], step)
    assert (y[rows * cols:] == 99).all() and float(scales[rows]) == 3.0


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_gated_rows(dev, pkg, dtype, cols):
    """gate and up side by side in the rows of one tensor."""
    rows = 1 if cols > 30000 else 5 if cols > 2000 else 20
    both = (2 * u.normal(u.gen(cols), (rows, 2 * cols))).to(u.TORCH[dtype])
    if rows > 3:
        both[3, cols:] = 0
    y, scales = call(pkg, dev, dtype, both, both[:, cols:], rows, cols, pitch=2 * cols)
    gate, up = both[:, :cols].double(), both[:, cols:].double()
    # exp to 2 units and its sum, quotient and product to half a unit in the last place each: 2^-22 and less of the value
    check(y[:rows * cols].view(rows, cols), scales[:rows], gate / (1 + torch.exp(-gate)) * up, 2.0 ** -21)
    assert (y[rows * cols:] == 99).all() and float(scales[rows]) == 3.0


@pytest.mark.parametrize("cols,pitch,off_x,off_y", [(64, 65, 0, 0), (64, 72, 1, 0), (64, 72, 0, 1), (64, 64, 0, 4), (1000, 1001, 3, 3), (4096, 5000, 8, 8), (9000, 9001, 1, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("gated", [False, True])
def test_pitches_and_offsets(dev, pkg, dtype, gated, cols, pitch, off_x, off_y):
    rows, g = 6, u.gen(cols)
    t = u.TORCH[dtype]
    raw = [u.normal(g, (rows * pitch + off_x,)).to(t) for _ in range(2)]
    x, up = (r[off_x:].view(rows, pitch) for r in raw)
    y, scales = torch.full((rows * cols + off_y + 8,), 99, dtype=torch.int8, device=u.GPU), torch.full((rows + 2,), 3.0, device=u.GPU)
    call(pkg, dev, dtype, x, up if gated else None, rows, cols, pitch, y[off_y:], scales[1:])
    v = x[:, :cols].double()
    if gated:
        v = v / (1 + torch.exp(-v)) * up[:, :cols].double()
    check(y[off_y:off_y + rows * cols].view(rows, cols), scales[1:rows + 1], v, 2.0 ** -21 if gated else 0.0)
    assert (y[:off_y] == 99).all() and (y[off_y + rows * cols:] == 99).all() and float(scales[0]) == 3.0 and float(scales[rows + 1]) == 3.0


@pytest.mark.parametrize("cols", [8, 100, 640, 5000, 40000])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_that_are_not_finite(dev, pkg, cols, gated, bad):
    """Their step is NaN, so that all of the row is; other rows are untouched by it."""
    x, up = (u.normal(u.gen(cols + i), (5, cols)).bfloat16() for i in range(2))
    clean = call(pkg, dev, "bf16", x, up if gated else None, 5, cols)
    (up if gated else x)[2, cols // 2] = bad
    y, scales = call(pkg, dev, "bf16", x, up if gated else None, 5, cols)
    assert torch.isnan(scales[:5]).tolist() == [False, False, True, False, False]
    keep = torch.tensor([0, 1, 3, 4], device=u.GPU)
    assert torch.equal(y[:5 * cols].view(5, cols)[keep], clean[0][:5 * cols].view(5, cols)[keep]) and torch.equal(scales[keep], clean[1][keep])


@pytest.mark.parametrize("value", [1e-45, 2e-44, 1e-38, 3e-36, 1e30, 3e38])
def test_smallest_and_largest_numbers(dev, pkg, value):
    """Steps that f32 hardly has, or whose reciprocal it has not: whole numbers stay within 127 and half a step (and a unit of the step) of the value."""
    x = torch.tensor([[0.0, 1.0, -1.0, 0.5, -0.25, 0.75, 0.1, -0.9]], device=u.GPU, dtype=torch.float64).mul(value).float()
    y, scales = call(pkg, dev, "f32", x, None, 1, 8)
    got, step = y[:8].double() * scales[:1].double(), float(scales[0])
    assert step > 0 and ((got - x[0].double()).abs() <= 0.5 * step + 127 * 2.0 ** -149 + 2.0 ** -22 * value).all()


def test_gates_far_below_and_above(dev, pkg):
    """exp(-x) overflows, or vanishes: 0 and x."""
    gate = torch.tensor([[-1000.0, -100.0, -90.0, 0.0, 100.0, 1000.0, 20.0, -20.0]], device=u.GPU)
    up = torch.ones_like(gate)
    y, scales = call(pkg, dev, "f32", gate, up, 1, 8)
    assert y[:8].tolist() == [0, 0, 0, 0, 13, 127, 3, 0] and float(scales[0]) == float(torch.tensor(1000.0) * torch.tensor(1 / 127.0))


def test_captured_and_replayed(dev, pkg):
    x = u.normal(u.gen(2), (7, 640)).bfloat16()
    y, scales = call(pkg, dev, "bf16", x, None, 7, 640)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        call(pkg, dev, "bf16", x, None, 7, 640, 0, y, scales)
    x.copy_(u.normal(u.gen(3), (7, 640)))
    graph.replay()
    q, step = u.quantise(x.float())
    assert torch.equal(y[:7 * 640].view(7, 640), q) and torch.equal(scales[:7], step)
