"""Cross attention over pages against the definition in 64 bits: tokens of any number against all positions of their sequence, of any number too, none among them."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu
# As tests/test_gpu_attention_paged.py: the same products, sums and roundings, without a diagonal.
REL = {"bf16": 6e-3, "f16": 8e-4}


class Encoded(u.Paged):
    """A paged cache of seqs = [(tokens, positions)], whatever the one has to do with the other."""

    def attend(self, q):
        hq, out = q.shape[1], torch.zeros(q.shape, dtype=torch.float64, device=u.GPU)
        for b, (new, n) in enumerate(self.seqs):
            if new == 0 or n == 0:
                continue
            at = slice(self.starts_h[b], self.starts_h[b + 1])
            k, v = (self.rows(w, b).repeat_interleave(hq // self.heads, 1) for w in range(2))
            s = torch.einsum("qhd,khd->hqk", q[at].double(), k) / self.d ** 0.5
            out[at] = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v)
        return out


def run(pkg, dev, cache, q):
    o = torch.full_like(q, 55.0)
    dev.attention_paged_cross(cache.view(), cache.batch(), u.codes(pkg.capi)[cache.dtype], q.shape[1], u.ptr(q), u.ptr(o), stream=u.stream())
    torch.cuda.synchronize()
    assert dev.status() == 0
    return o


def check(cache, q, o):
    used = cache.starts_h[-1]
    assert (o[used:] == 55).all()
    want, got = cache.attend(q)[:used], o[:used].double()
    assert torch.isfinite(got).all()
    for b, (new, n) in enumerate(cache.seqs):
        at = slice(cache.starts_h[b], cache.starts_h[b + 1])
        if new == 0:
            continue
        if n == 0:
            assert (got[at] == 0).all()
            continue
        off = (got[at] - want[at]).norm() / want[at].norm()
        assert off <= REL[cache.dtype], (b, cache.seqs[b], float(off))
        worst = ((got[at] - want[at]).abs().amax(-1) / want[at].square().mean(-1).sqrt()).max()
        assert worst <= 12 * REL[cache.dtype], (b, cache.seqs[b], float(worst))


def one(pkg, dev, seed, seqs, hq, hkv, d, page, dtype, held, **more):
    cache = Encoded(pkg, seed, seqs, hkv, d, page, dtype, held, **more)
    q = u.normal(u.gen(seed + 1), (cache.tokens, hq, d), 1.5).to(u.TORCH[dtype])
    check(cache, q, run(pkg, dev, cache, q))


TYPES = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "i8"), ("f16", "i8")]


@pytest.mark.parametrize("dtype,held", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (3, 3), (14, 2), (20, 1)])
def test_single_tokens(dev, pkg, dtype, held, d, hq, hkv):
    one(pkg, dev, 11, [(1, n) for n in (1, 0, 2, 15, 16, 17, 31, 64, 0, 129, 700, 3001)], hq, hkv, d, 16, dtype, held)


@pytest.mark.parametrize("dtype,held", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (2, 2), (14, 2), (20, 1)])
def test_prompts(dev, pkg, dtype, held, d, hq, hkv):
    """More tokens than positions and fewer, sequences without either."""
    one(pkg, dev, 12, [(300, 1), (0, 77), (130, 130), (3, 500), (257, 1000), (0, 0), (1, 1), (64, 0), (31, 2000), (500, 60)], hq, hkv, d, 32, dtype, held, slack=2, gap=5)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 96, 128, 1000, 4096])
@pytest.mark.parametrize("held", ["bf16", "i8"])
def test_page_sizes(dev, pkg, page, held):
    one(pkg, dev, 13, [(1, 515), (200, 44), (12, 12), (1, page), (1, page + 1), (70, 1025)], 8, 2, 128, page, "bf16", held)


@pytest.mark.parametrize("held", ["bf16", "i8"])
@pytest.mark.parametrize("new", [1, 200])
def test_all_empty(dev, pkg, held, new):
    one(pkg, dev, 14, [(new, 0)] * 200, 8, 2, 64, 16, "bf16", held)


@pytest.mark.parametrize("batch", [1, 150, 700])
@pytest.mark.parametrize("held", ["f16", "i8"])
def test_many_sequences(dev, pkg, batch, held):
    one(pkg, dev, 16, [(1 + i % 3, 37 * i % 211) for i in range(1, batch + 1)], 8, 4, 128, 16, "f16", held)


def test_long(dev, pkg):
    one(pkg, dev, 15, [(1, 40000)], 8, 2, 128, 64, "bf16", "bf16")
    one(pkg, dev, 15, [(700, 9000), (1, 20000)], 4, 2, 64, 64, "bf16", "i8")


def test_infinities_in_places_no_sequence_has(dev, pkg):
    for junk in (float("inf"), -float("inf"), 6e4):
        for held in ("f16", "i8"):
            one(pkg, dev, 17, [(1, 70), (40, 90), (90, 3)], 8, 2, 128, 16, "f16", held, junk=junk)


def test_one_key_takes_all(dev, pkg):
    """Keys far apart, whichever token asks: V of the chosen one, before and behind the token's own number."""
    cache = Encoded(pkg, 18, [(150, 150)], 1, 64, 16, "bf16", "bf16")
    for i in range(150):
        row = torch.zeros(64, device=u.GPU)
        row[0], row[1] = i * 2.0, -(i * i) / 64.0
        cache.kv[0][int(cache.table[0, i // 16]), 0, i % 16] = row.bfloat16()
    # keys rounded to bf16: the definition says which one each token picks
    q = torch.zeros((150, 1, 64), dtype=torch.bfloat16, device=u.GPU)
    q[:, 0, 0] = torch.arange(150, device=u.GPU).flip(0).bfloat16() * 16
    q[:, 0, 1] = 512.0
    o, want = run(pkg, dev, cache, q), cache.attend(q)
    s = torch.einsum("qhd,khd->hqk", q.double(), cache.rows(0, 0)) / 8
    top = s[0].topk(2).values
    sure = top[:, 0] - top[:, 1] > 25
    # The largest weight is 2^x with x up to 8, taken against a maximum that may lag, and is rounded to bf16 (2^-8 of it at most) while the sum is of unrounded ones; the
    # result is rounded once more.  The other keys weigh e^-25 each.
    assert int(sure.sum()) > 20 and ((o[sure].double() - want[sure]).abs() <= 2.02 * u.HALF_ULP["bf16"] * want[sure].abs() + 1e-8).all()


def test_results_do_not_depend_on_the_run_or_the_stream(dev, pkg):
    cache = Encoded(pkg, 21, [(1, 5000), (200, 3000), (1, 20), (9, 0)], 4, 128, 16, "bf16", "i8")
    q = u.normal(u.gen(22), (cache.tokens, 16, 128)).bfloat16()
    first = run(pkg, dev, cache, q)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(5):
            assert torch.equal(run(pkg, dev, cache, q), first)


@pytest.mark.parametrize("new", [1, 40])
def test_in_a_graph(dev, pkg, new):
    cache = Encoded(pkg, 23, [(new, 900), (new, 300)], 2, 128, 16, "bf16", "bf16", junk=0.0)
    q = u.normal(u.gen(24), (2 * new, 8, 128)).bfloat16()
    o = run(pkg, dev, cache, q)
    view, batch = cache.view(), cache.batch()
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=s):
        dev.attention_paged_cross(view, batch, pkg.capi.BF16, 8, u.ptr(q), u.ptr(o), stream=torch.cuda.current_stream().cuda_stream)
    for lens in ((900, 300), (17, 0), (0, 299)):
        cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        cache.seqs = [(new, n) for n in lens]
        o.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert dev.status() == 0
        check(cache, q, o)


@pytest.mark.parametrize("held", ["bf16", "i8"])
def test_what_is_outside_is_reported(dev, pkg, held):
    def page(c):
        c.table[1, 1] = c.pages + 5

    def length(c):
        c.lens[1] = c.pitch * c.page + 1

    def negative(c):
        c.lens[1] = -1

    for spoil in (page, length, negative):
        for news in ((1, 1, 1), (4, 4, 4), (30, 4, 40)):
            c = Encoded(pkg, 3, [(news[0], 80), (news[1], 60), (news[2], 0)], 2, 64, 16, "bf16", held)
            spoil(c)
            q = u.normal(u.gen(4), (c.tokens, 4, 64)).bfloat16()
            o = torch.full_like(q, 55.0)
            dev.attention_paged_cross(c.view(), c.batch(), pkg.capi.BF16, 4, u.ptr(q), u.ptr(o), stream=u.stream())
            with pytest.raises(pkg.hal.KernelError, match="left it out"):
                pkg.hal.check(pkg.capi.lib().tsm100_stream_synchronize(dev._h, None))
            if spoil is not page:
                assert (o[c.starts_h[1]:c.starts_h[2]] == 55).all()
            c.seqs = [c.seqs[0], (0, 0), c.seqs[2]]
            want = c.attend(q)
            at = slice(0, c.starts_h[1])
            assert (o[at].double() - want[at]).norm() <= REL["bf16"] * want[at].norm(), (spoil.__name__, news)
            assert (o[c.starts_h[2]:] == 0).all()
            assert dev.status() == 0


@pytest.mark.parametrize("held", ["bf16", "i8"])
@pytest.mark.parametrize("news,group,page", [((1, 1, 1), 4, 16), ((3, 1, 0), 4, 16), ((3, 40, 9), 4, 16), ((3, 40, 9), 5, 3)])
def test_any_number_of_new_tokens_allowed(dev, pkg, news, group, page, held):
    """max_new as large as it goes takes no memory by itself: the same result, bit for bit, as with the call's tokens."""
    cache = Encoded(pkg, 31, list(zip(news, (90, 700, 33))), 2, 64, page, "bf16", held)
    q = u.normal(u.gen(32), (cache.tokens, 2 * group, 64)).bfloat16()
    got = []
    for most in (cache.tokens, 2**31 - 1):
        batch = pkg.hal.PagedBatch(3, cache.tokens, most, 0, cache.pitch, u.ptr(cache.table), u.ptr(cache.lens), u.ptr(cache.starts))
        o = torch.full_like(q, 55.0)
        dev.attention_paged_cross(cache.view(), batch, pkg.capi.BF16, 2 * group, u.ptr(q), u.ptr(o), stream=u.stream())
        torch.cuda.synchronize()
        assert dev.status() == 0
        got.append(o)
    assert torch.equal(*got)
    check(cache, q, got[0])


def test_refusals(dev, pkg):
    capi, hal = pkg.capi, pkg.hal
    x = torch.zeros(4096, device=u.GPU)
    p = x.data_ptr()

    def bad(match, dtype=capi.BF16, heads_q=4, cache=None, q=p, o=p):
        kv = dict(dtype=capi.BF16, heads_kv=2, head_dim=64, page_size=16, pages=2, k=p, v=p) | (cache or {})
        with pytest.raises(hal.KernelError, match="attention_paged_cross: .*" + match):
            dev.attention_paged_cross(hal.PagedKv(**kv), hal.PagedBatch(1, 1, 1, 0, 1, p, p, p), dtype, heads_q, q, o, stream=u.stream())

    bad("dtype must be", dtype=capi.F32)
    bad("must hold", cache={"dtype": capi.F16})
    bad("head_dim must be 64 or 128", cache={"head_dim": 96})
    bad("multiple of heads_kv", heads_q=3)
    bad("null buffer", q=0)
    bad("16-byte aligned", o=p + 2)
    dev.attention_paged_cross(hal.PagedKv(capi.BF16, 2, 64, 16, 2, p, p), hal.PagedBatch(0, 0, 0, 0, 0, 0, 0, 0), capi.BF16, 4, 0, 0, stream=u.stream())
