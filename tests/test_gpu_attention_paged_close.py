"""Attention over pages, as near to the definition as its roundings allow and no farther: one of the probabilities and one of the output, and nothing for turning an 8-bit
cache's numbers into the type.

A rounding to b significant bits is off by 2^-b / sqrt 3 of a number at the foot of its binade, in the root mean square over a binade 0.74 times that: 2.1e-4 for f16,
1.7e-3 for bf16.  Errors of terms of either sign add up as the terms do, so each rounding counts alike in the norm of many outputs: sqrt 2 times that where probabilities have the
output's type; probabilities in f16 under a bf16 output count nothing.  A third rounding would be another 22 %, of K and V both 41 %.  15 % is allowed."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu
ROUNDING = {"f16": 2.0 ** -11 / 3 ** 0.5 * 0.7355, "bf16": 2.0 ** -8 / 3 ** 0.5 * 0.7355}


@pytest.mark.parametrize("dtype,held", [("f16", "i8"), ("bf16", "i8"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 90])
def test_two_roundings(dev, pkg, new, d, dtype, held):
    seqs = [(new, n) for n in (500, 777, 1900, 4000, 640, 2300)]
    cache = u.Paged(pkg, 61, seqs, 4, d, 16, dtype, held)
    q = u.normal(u.gen(62), (cache.tokens, 16, d)).to(u.TORCH[dtype])
    o = torch.zeros_like(q)
    dev.attention_paged(cache.view(), cache.batch(), u.codes(pkg.capi)[dtype], 16, u.ptr(q), u.ptr(o), stream=u.stream())
    want = cache.attend(q)
    off = float((o.double() - want).norm() / want.norm())
    count = 1 if (dtype, held) == ("bf16", "i8") else 2
    assert off <= 1.15 * count ** 0.5 * ROUNDING[dtype], (off, off / ROUNDING[dtype])
    assert dev.status() == 0
