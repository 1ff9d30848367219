"""Keys that are not finite: softmax of a row with a NaN or +inf among the scores that it sees is NaN, of one with -inf it is that of the others.  Wherever in a tile of
keys they lie, and whether a row has its softmax from one kernel or another."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")
REL = {"bf16": 6e-3, "f16": 8e-4}  # what the attention of finite inputs is held to


def spoil(rows, kind):
    """rows [..., d] of keys: NaN; or 0 but for the first number, +inf."""
    if kind == "nan":
        rows[..., 3] = NAN
    else:
        rows[:] = 0
        rows[..., 0] = INF


def queries(g, shape, dtype, kind):
    q = u.normal(g, shape)
    q[..., 0] = {"nan": 1.0, "+inf": 0.75, "-inf": -0.75}[kind]
    return q.to(u.TORCH[dtype])


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,held,kind", [("bf16", "bf16", "nan"), ("f16", "f16", "nan"), ("bf16", "i8", "nan"), ("f16", "i8", "nan"), ("bf16", "bf16", "+inf"),
                                             ("f16", "f16", "+inf"), ("bf16", "bf16", "-inf"), ("f16", "f16", "-inf")])
def test_paged(dev, pkg, new, d, dtype, held, kind):
    """Sequence b has such a key at position 225 + b of 300, in its first head only: all columns of a tile of 16 or 32, before the new tokens and among them."""
    at = [225 + b for b in range(48)]
    cache = u.Paged(pkg, 31, [(new, 300)] * len(at), 2, d, 16, dtype, held)
    for b, pos in enumerate(at):
        page, place = int(cache.table[b, pos // 16]), pos % 16
        if held == "i8":
            cache.scales[0][page, 0, place] = NAN
        else:
            spoil(cache.kv[0][page, 0, place], kind)
    q = queries(u.gen(32), (cache.tokens, 8, d), dtype, kind)
    o = torch.zeros_like(q)
    dev.attention_paged(cache.view(), cache.batch(), u.codes(pkg.capi)[dtype], 8, u.ptr(q), u.ptr(o), stream=u.stream())
    want = cache.attend(q)
    for b, pos in enumerate(at):
        first = cache.starts_h[b]
        for r in range(new):
            sees = pos <= 300 - new + r
            if sees and kind != "-inf":
                assert torch.isnan(o[first + r, :4]).all(), (b, r)
        rows = slice(first, first + new)
        ok = ~torch.isnan(want[rows])
        assert torch.equal(ok, ~torch.isnan(o[rows])), b
        assert (o[rows].double() - want[rows])[ok].norm() <= REL[dtype] * want[rows][ok].norm(), b
    assert dev.status() == 0


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kind", ["nan", "+inf"])
def test_plain(dev, pkg, causal, d, dtype, kind):
    """Head b has such a key at position 100 + b of 320."""
    heads, seq = 36, 320
    g, t = u.gen(33), u.TORCH[dtype]
    k, v = (u.normal(g, (heads, seq, d)).to(t) for _ in range(2))
    for b in range(heads):
        spoil(k[b, 100 + b], kind)
    q = queries(g, (heads, seq, d), dtype, kind)
    o = torch.zeros_like(q)
    dev.attention(u.codes(pkg.capi)[dtype], 1, heads, heads, seq, d, u.ptr(q), u.ptr(k), u.ptr(v), u.ptr(o), causal=causal, stream=u.stream())
    for b in range(heads):
        first = 100 + b if causal else 0
        assert torch.isnan(o[b, first:]).all() and torch.isfinite(o[b, :first]).all(), b
    assert dev.status() == 0
