"""Attention over pages against the definition in 64 bits: single tokens and chunks side by side, sequences without tokens, pages that end inside tiles,
groups of every size, caches of 16 and 8 bits, NaN wherever a sequence has no position."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu
# Inputs are N(0, 1) with rows scaled by exp(N(0, 0.5)).  The output is rounded once (2^-9 of it at most, bf16; a third of that root mean square), the
# probabilities may be, and the 8-bit cache's values as they turn into the type: three roundings more of 1.1e-3 each in the mean.  f16: an eighth.
REL = {"bf16": 6e-3, "f16": 8e-4}


def run(pkg, dev, cache, q, max_len=0):
    o = torch.full_like(q, 55.0)
    dev.attention_paged(cache.view(), cache.batch(max_len=max_len), u.codes(pkg.capi)[cache.dtype], q.shape[1], u.ptr(q), u.ptr(o), stream=u.stream())
    torch.cuda.synchronize()
    assert dev.status() == 0
    return o


def check(cache, q, o):
    used = cache.starts_h[-1]
    assert (o[used:] == 55).all()
    want, got = cache.attend(q)[:used], o[:used].double()
    assert torch.isfinite(got).all()
    for b in range(len(cache.seqs)):  # sequence by sequence, so that none hides behind a longer one
        at = slice(cache.starts_h[b], cache.starts_h[b + 1])
        if at.start == at.stop:
            continue
        off = (got[at] - want[at]).norm() / want[at].norm()
        assert off <= REL[cache.dtype], (b, cache.seqs[b], float(off))
        worst = ((got[at] - want[at]).abs().amax(-1) / want[at].square().mean(-1).sqrt()).max()
        assert worst <= 12 * REL[cache.dtype], (b, cache.seqs[b], float(worst))


def one(pkg, dev, seed, seqs, hq, hkv, d, page, dtype, held, **more):
    cache = u.Paged(pkg, seed, seqs, hkv, d, page, dtype, held, **more)
    q = u.normal(u.gen(seed + 1), (cache.tokens, hq, d), 1.5).to(u.TORCH[dtype])
    check(cache, q, run(pkg, dev, cache, q))


@pytest.mark.parametrize("dtype,held", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "i8"), ("f16", "i8")])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (1, 1), (14, 2), (20, 1)])
def test_single_tokens(dev, pkg, dtype, held, d, hq, hkv):
    """One new token each: lengths of one, inside and at the end of pages and tiles, long ones that several CTAs share."""
    one(pkg, dev, 11, [(1, n) for n in (1, 2, 15, 16, 17, 31, 64, 65, 129, 700, 3001)], hq, hkv, d, 16, dtype, held)


@pytest.mark.parametrize("dtype,held", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "i8"), ("f16", "i8")])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (2, 2), (14, 2), (20, 1)])
def test_mixed(dev, pkg, dtype, held, d, hq, hkv):
    one(pkg, dev, 12, [(1, 300), (0, 77), (130, 130), (3, 500), (257, 1000), (0, 0), (1, 1), (64, 128), (31, 2000)], hq, hkv, d, 32, dtype, held, slack=2, gap=5)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 48, 64, 96, 128, 256, 1000])
@pytest.mark.parametrize("held", ["bf16", "i8"])
def test_page_sizes(dev, pkg, page, held):
    one(pkg, dev, 13, [(1, 515), (200, 444), (12, 12), (1, page), (1, page + 1), (70, 1025)], 8, 2, 128, page, "bf16", held)


@pytest.mark.parametrize("held", ["bf16", "i8"])
@pytest.mark.parametrize("d", [64, 128])
def test_long(dev, pkg, held, d):
    one(pkg, dev, 14, [(1, 40000)], 8, 2, d, 64, "bf16", held)
    one(pkg, dev, 15, [(500, 9000), (1, 20000)], 4, 2, d, 64, "bf16", held)


@pytest.mark.parametrize("batch", [1, 2, 150, 700])
@pytest.mark.parametrize("held", ["f16", "i8"])
def test_many_sequences(dev, pkg, batch, held):
    one(pkg, dev, 16, [(1, 1 + 37 * i % 211) for i in range(batch)], 8, 4, 128, 16, "f16", held)


def test_infinities_in_places_no_sequence_has(dev, pkg):
    for junk in (float("inf"), -float("inf"), 6e4):
        for held in ("f16", "i8"):
            one(pkg, dev, 17, [(1, 70), (40, 90), (1, 3)], 8, 2, 128, 16, "f16", held, junk=junk)


def test_a_token_sees_itself_and_no_later_one(dev, pkg):
    """Keys so far apart that each row's softmax is its own position: row i gives V[i] bit for bit."""
    cache = u.Paged(pkg, 18, [(150, 150)], 1, 64, 16, "bf16", "bf16")
    at = torch.arange(150, device=u.GPU)
    rows = torch.zeros((150, 64), device=u.GPU)
    rows[:, 0] = at * 8.0
    for i in range(150):
        cache.kv[0][int(cache.table[0, i // 16]), 0, i % 16] = rows[i].bfloat16()
    q = torch.zeros((150, 1, 64), dtype=torch.bfloat16, device=u.GPU)
    q[..., 0] = 64.0
    o = run(pkg, dev, cache, q)
    assert torch.equal(o[:, 0], cache.rows(1, 0)[:, 0].bfloat16())


def test_extreme_scores(dev, pkg):
    """Scores of +-1e4 and rows of equal ones."""
    cache = u.Paged(pkg, 19, [(1, 333), (90, 200)], 2, 128, 16, "bf16", "bf16")
    q = u.normal(u.gen(20), (cache.tokens, 4, 128), 600.0).bfloat16()
    q[0] = 0
    o = run(pkg, dev, cache, q)
    want = cache.attend(q)
    assert torch.isfinite(o).all()
    assert (o[0].double() - want[0]).norm() <= REL["bf16"] * want[0].norm()
    # where one key takes all but a millionth, the output is that key's V
    k = cache.rows(0, 1).repeat_interleave(2, 1)
    for r in range(90):
        s = torch.einsum("hd,khd->hk", q[1 + r].double(), k[:111 + r]) / 128 ** 0.5
        top = s.topk(2).values
        sure = top[:, 0] - top[:, 1] > 25
        assert ((o[1 + r].double() - want[1 + r]).abs().amax(-1)[sure] <= 2.0 ** -8 * want[1 + r].abs().amax(-1)[sure]).all()


def test_results_do_not_depend_on_the_run_or_the_stream(dev, pkg):
    cache = u.Paged(pkg, 21, [(1, 5000), (200, 3000), (1, 20)], 4, 128, 16, "bf16", "i8")
    q = u.normal(u.gen(22), (cache.tokens, 16, 128)).bfloat16()
    first = run(pkg, dev, cache, q)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(5):
            assert torch.equal(run(pkg, dev, cache, q), first)
    assert torch.equal(run(pkg, dev, cache, q, max_len=5000), first)


def test_in_a_graph(dev, pkg):
    """Captured once, replayed for other lengths: the arrays are read when the kernels run."""
    cache = u.Paged(pkg, 23, [(1, 900), (1, 300)], 2, 128, 16, "bf16", "bf16", junk=0.0)
    q = u.normal(u.gen(24), (2, 8, 128)).bfloat16()
    o = torch.zeros_like(q)
    view, batch = cache.view(), cache.batch(max_len=900)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        dev.attention_paged(view, batch, pkg.capi.BF16, 8, u.ptr(q), u.ptr(o), stream=s.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        dev.attention_paged(view, batch, pkg.capi.BF16, 8, u.ptr(q), u.ptr(o), stream=torch.cuda.current_stream().cuda_stream)
    for lens in ((900, 300), (17, 1), (512, 299)):
        cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        cache.seqs = [(1, n) for n in lens]
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert dev.status() == 0
        want = cache.attend(q)
        assert (o.double() - want).norm() <= REL["bf16"] * want.norm()


@pytest.mark.parametrize("held", ["bf16", "i8"])
def test_what_is_outside_is_reported(dev, pkg, held):
    """The other sequences are served all the same."""
    def page(c):
        c.table[1, 1] = c.pages + 5

    def negative(c):
        c.table[1, 0] = -1

    def length(c):
        c.lens[1] = c.pitch * c.page + 1

    def short(c):
        c.lens[1] = 3

    for spoil in (page, negative, length, short):
        for news in ((1, 1, 1), (4, 4, 4), (30, 4, 40)):
            c = u.Paged(pkg, 3, [(news[0], 80), (news[1], 60), (news[2], 70)], 2, 64, 16, "bf16", held)
            if spoil is short and news[1] == 1:
                c.lens[1] = 0
            else:
                spoil(c)
            q = u.normal(u.gen(4), (c.tokens, 4, 64)).bfloat16()
            o = torch.zeros_like(q)
            dev.attention_paged(c.view(), c.batch(), pkg.capi.BF16, 4, u.ptr(q), u.ptr(o), stream=u.stream())
            with pytest.raises(pkg.hal.KernelError, match="left it out"):
                pkg.hal.check(pkg.capi.lib().tsm100_stream_synchronize(dev._h, None))
            c.seqs = [c.seqs[0], (0, 0), c.seqs[2]]
            want = c.attend(q)
            for b in (0, 2):
                at = slice(c.starts_h[b], c.starts_h[b + 1])
                assert (o[at].double() - want[at]).norm() <= REL["bf16"] * want[at].norm(), (spoil.__name__, news, b)
            assert dev.status() == 0


def test_refusals(dev, pkg):
    capi, hal = pkg.capi, pkg.hal
    x = torch.zeros(4096, device=u.GPU)
    p = x.data_ptr()

    def bad(match, dtype=capi.BF16, heads_q=4, cache=None, q=p, o=p):
        kv = dict(dtype=capi.BF16, heads_kv=2, head_dim=64, page_size=16, pages=2, k=p, v=p) | (cache or {})
        b = hal.PagedBatch(1, 1, 1, 0, 1, p, p, p)
        with pytest.raises(hal.KernelError, match=match):
            dev.attention_paged(hal.PagedKv(**kv), b, dtype, heads_q, q, o, stream=u.stream())

    bad("dtype must be", dtype=capi.F32)
    bad("must hold", cache={"dtype": capi.F16})
    bad("head_dim must be 64 or 128", cache={"head_dim": 96})
    bad("multiple of heads_kv", heads_q=3)
    bad("multiple of heads_kv", heads_q=0)
    bad("null buffer", q=0)
    bad("16-byte aligned", o=p + 2)
    dev.attention_paged(hal.PagedKv(capi.BF16, 2, 64, 16, 2, p, p), hal.PagedBatch(0, 0, 0, 0, 0, 0, 0, 0), capi.BF16, 4, 0, 0, stream=u.stream())
