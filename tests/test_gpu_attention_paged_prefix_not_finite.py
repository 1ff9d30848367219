"""Keys and values that are not finite behind and in a shared prefix, and in cross attention, where records come from tcgen05 as well as from the kernel for few rows."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402
from test_gpu_attention_paged_prefix import Sharing, check, run  # noqa: E402

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")

# sequences, page, pages of the prefix: the prefix and the rest in one stream; the prefix on tcgen05 (440 rows of a KV head on 8192 positions: route.hpp says so of
# each case here, see below); both on tcgen05 beside single tokens
FORMS = {"stream": ([(1, 40)] * 3, 16, 4), "prefix_on_tcgen05": ([(1, 40)] * 110, 64, 128), "both_on_tcgen05": ([(1, 40)] * 30 + [(60, 60), (100, 400)], 64, 128)}


def caches(pkg, form, held="bf16", d=128):
    # route.hpp: prefix_on_tcgen05
    seqs, page, shared = FORMS[form]
    passes, size = -(-sum(new for new, _ in seqs) * 4 // 16), 2 * shared * page * 4 * d * (1 if held == "i8" else 2)
    assert ((passes - 1) * size > (200 << 20 if held == "i8" else 80 << 20)) == (form != "stream")
    cache = Sharing(pkg, 51, seqs, 4, d, page, "bf16", held, shared, junk=0.0 if held != "i8" else NAN)
    q = u.normal(u.gen(52), (cache.tokens, 16, d)).abs().bfloat16() + 0.5
    return cache, q


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("spoilt", [(True, False), (False, True), (True, True)])
def test_parts_whose_scores_are_all_minus_infinity(dev, pkg, form, d, spoilt):
    """They weigh nothing beside the other part; both: NaN, as of one softmax over all of them."""
    cache, q = caches(pkg, form, d=d)
    shared = torch.zeros(cache.pages, dtype=torch.bool, device=u.GPU)
    shared[cache.prefix.long()] = True
    for part, pages in enumerate((shared, ~shared)):
        if spoilt[part]:
            cache.kv[0][pages, :, :, 0] = -INF
    o = run(pkg, dev, cache, q)
    if all(spoilt):
        assert torch.isnan(o).all()
    else:
        check(cache, q, o)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("held,kind", [("bf16", "nan"), ("bf16", "inf"), ("i8", "nan")])
def test_keys(dev, pkg, form, held, kind):
    """A NaN or +inf score in the prefix makes NaN of all rows of its KV head; in the middle of a sequence's own positions, of the tokens from there on."""
    for in_prefix in (True, False):
        cache, q = caches(pkg, form, held)
        b = len(cache.seqs) - 1
        new, n = cache.seqs[b]
        pos = 70 % (cache.shared * cache.page) if in_prefix else n - (new + 1) // 2
        page, place = int(cache.table[b, pos // cache.page]), pos % cache.page
        if held == "i8":
            cache.scales[0][page, 1, place] = NAN
        else:
            cache.kv[0][page, 1, place, 0] = NAN if kind == "nan" else INF
        o = run(pkg, dev, cache, q)
        gone = torch.isnan(o).all(-1)
        want = torch.zeros_like(gone)
        if in_prefix:
            want[:, 4:8] = True
        else:
            want[cache.starts_h[b] + pos - (n - new):cache.starts_h[b + 1], 4:8] = True
        assert torch.equal(gone, want) and torch.isfinite(o[~gone]).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("held", ["bf16", "i8"])
def test_values(dev, pkg, form, held):
    """A value that is not finite reaches its column (8 bits: its row's step, so all columns) of the tokens that see it, perhaps of earlier tokens of its sequence in the call, whose weight for it is 0,
    and nobody else: other sequences and heads keep their bits."""
    for in_prefix in (True, False):
        cache, q = caches(pkg, form, held)
        clean = run(pkg, dev, cache, q)
        b = len(cache.seqs) - 1
        new, n = cache.seqs[b]
        pos = 70 % (cache.shared * cache.page) if in_prefix else n - (new + 1) // 2
        page, place = int(cache.table[b, pos // cache.page]), pos % cache.page
        columns = slice(None) if held == "i8" else slice(9, 10)
        if held == "i8":
            cache.scales[1][page, 1, place] = NAN
        else:
            cache.kv[1][page, 1, place, 9] = NAN
        o = run(pkg, dev, cache, q)
        first, last = (0, cache.tokens) if in_prefix else (cache.starts_h[b], cache.starts_h[b + 1])
        sees = 0 if in_prefix else cache.starts_h[b] + pos - (n - new)
        assert torch.isnan(o[sees:last, 4:8, columns]).all()
        o[first:last, 4:8, columns] = clean[first:last, 4:8, columns]
        assert torch.equal(o, clean)
