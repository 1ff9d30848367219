"""Attention over pages where what counts is small beside something that does not: a first key that takes almost all the weight and says nothing, values far larger than
those a row sees or weighs.  Against the definition in 64 bits.

Bounds.  A probability is rounded to f16 (8-bit and f16 caches; f16 has numbers to 2^-14 in full) and the output to its type; each rounding is uniform within half a unit in
the last place, so its root mean square is that over sqrt 3 of what it rounds at most, and rounding errors of terms of either sign add up as the terms themselves do.
Together sqrt 2 * 2^-11 / sqrt 3 = 4.0e-4 of the output's norm for f16 and 2^-8 / sqrt 3 = 2.3e-3 for bf16 (its output's rounding alone); f32 sums and exponentials are 1e-6.
Half as much again is allowed."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu
REL = {"f16": 6e-4, "bf16": 3.5e-3}


def caches(pkg, seqs, d, dtype, held, group, seed):
    """Keys whose first number is 0, small besides; queries whose first number is 8.  Values N(0, 1) times 64."""
    cache = u.Paged(pkg, seed, seqs, 2, d, 16, dtype, held, junk=1.0)
    g = u.gen(seed + 1)
    if held == "i8":
        cache.kv[0].copy_(torch.randint(-20, 21, cache.kv[0].shape, generator=g, device=u.GPU, dtype=torch.int8))
        cache.kv[0][..., 0] = 0
        cache.scales[0].fill_(1 / 64)
        cache.kv[1].copy_(torch.randint(-127, 128, cache.kv[1].shape, generator=g, device=u.GPU, dtype=torch.int8))
        cache.scales[1].fill_(1.0)
    else:
        cache.kv[0].copy_(u.normal(g, cache.kv[0].shape, 0.2))
        cache.kv[0][..., 0] = 0
        cache.kv[1].copy_(u.normal(g, cache.kv[1].shape, 64.0))
    q = u.normal(g, (cache.tokens, 2 * group, d)).to(u.TORCH[dtype])
    q[..., 0] = 8
    return cache, q


def put_key(cache, b, pos, first, d):
    """The key at a position gets the score first * 8 / sqrt d from its first number and nothing from the others."""
    page, place = int(cache.table[b, pos // 16]), pos % 16
    cache.kv[0][page, :, place] = 0
    if cache.cache == "i8":
        cache.kv[0][page, :, place, 0] = 127 if first > 0 else -127
        cache.scales[0][page, :, place] = abs(first) / 127
    else:
        cache.kv[0][page, :, place, 0] = first
    return page, place


def check(dev, pkg, cache, q, dtype):
    o = torch.zeros_like(q)
    dev.attention_paged(cache.view(), cache.batch(), u.codes(pkg.capi)[dtype], q.shape[1], u.ptr(q), u.ptr(o), stream=u.stream())
    torch.cuda.synchronize()
    assert dev.status() == 0
    want = cache.attend(q)
    for b in range(len(cache.seqs)):
        at = slice(cache.starts_h[b], cache.starts_h[b + 1])
        off = float((o[at].double() - want[at]).norm() / want[at].norm())
        assert off <= REL[dtype], (b, off)


# one token: a tile of few rows; three: of sixteen; forty: a chunk's.  bf16 caches hold probabilities in bf16, which has no such end
FORMS = [("f16", "i8"), ("bf16", "i8"), ("f16", "f16")]


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,held", FORMS)
def test_a_first_key_that_takes_almost_all_weight(dev, pkg, new, d, dtype, held):
    cache, q = caches(pkg, [(new, 8000), (new, 3000)], d, dtype, held, 4, 41)
    for b in range(2):
        page, place = put_key(cache, b, 0, 14.0 * d ** 0.5 / 8, d)  # e^14: 2^20 times the others' weight
        cache.kv[1][page, :, place] = 0
    check(dev, pkg, cache, q, dtype)


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,held", FORMS[:2])
def test_one_value_far_larger_that_weighs_nothing(dev, pkg, new, d, dtype, held):
    """65536 times the others' step, behind a score 40 below theirs; at the beginning, in the middle, and in every tile of the first half."""
    for positions in ([2], [700], range(5, 700, 16)):
        cache, q = caches(pkg, [(new, 1500), (new, 720 + new)], d, dtype, held, 4, 43)
        for b in range(2):
            for pos in positions:
                page, place = put_key(cache, b, pos, -40.0 * d ** 0.5 / 8, d)
                cache.scales[1][page, :, place] = 65536.0
        check(dev, pkg, cache, q, dtype)


@pytest.mark.parametrize("new", [3, 40])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,held", FORMS[:2])
def test_one_value_far_larger_that_most_rows_do_not_see(dev, pkg, new, d, dtype, held):
    cache, q = caches(pkg, [(new, 1500)], d, dtype, held, 4, 45)
    cache.scales[1][int(cache.table[0, 1499 // 16]), :, 1499 % 16] = 65536.0
    o = torch.zeros_like(q)
    dev.attention_paged(cache.view(), cache.batch(), u.codes(pkg.capi)[dtype], q.shape[1], u.ptr(q), u.ptr(o), stream=u.stream())
    want = cache.attend(q)
    assert dev.status() == 0
    for at in (slice(0, new - 1), slice(new - 1, new)):
        off = float((o[at].double() - want[at]).norm() / want[at].norm())
        assert off <= REL[dtype], (at, off)
