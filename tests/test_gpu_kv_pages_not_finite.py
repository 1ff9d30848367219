"""NaN and infinities on their way through an 8-bit cache: max|x| / 127 is none then, so the row's step is not finite and the row is NaN when it is read; rows beside it
keep their numbers."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,d", [(2, 16), (3, 64), (2, 128), (1, 240)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("which", [0, 1])
def test_a_row_that_is_not_finite_stays_so(dev, pkg, dtype, heads, d, bad, which):
    cache = u.Paged(pkg, 7, [(40, 60), (1, 5)], heads, d, 16, dtype, "i8", junk=1.0)
    g, t = u.gen(8), u.TORCH[dtype]
    new = [u.normal(g, (cache.tokens, heads, d)).to(t) for _ in range(2)]
    clean = [x.clone() for x in new]
    spots = [(token, token % heads, (token * 7) % d) for token in (0, 3, 17, 39, 40)]  # in every lane of a row and at both ends of the sequences
    for token, head, at in spots:
        new[which][token, head, at] = bad
    new[which][9, 0] = bad  # a row of nothing else
    spots.append((9, 0, 0))
    code = u.codes(pkg.capi)[dtype]
    dev.kv_page_append(cache.view(), cache.batch(), code, u.ptr(new[0]), u.ptr(new[1]), stream=u.stream())
    out = [torch.zeros((cache.tokens, heads, d), dtype=t, device=u.GPU) for _ in range(2)]
    dev.kv_page_read(cache.view(), cache.batch(), code, u.ptr(out[0]), u.ptr(out[1]), stream=u.stream())
    for w in range(2):
        q, step = u.quantise(clean[w].float())
        want = (q.float() * step[..., None]).to(t)
        if w == which:
            for token, head, _ in spots:
                assert torch.isnan(out[w][token, head]).all(), (token, head)
                want[token, head] = 0
                out[w][token, head] = 0
        assert torch.equal(out[w], want)
    assert dev.status() == 0
