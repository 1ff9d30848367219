"""Attention of sequences that begin with the same pages against the definition in 64 bits, and against attention_paged on the same pages."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu
# As tests/test_gpu_attention_paged.py: the two parts of a row are joined in f32, which rounds nothing that counts beside the probabilities.
REL = {"bf16": 6e-3, "f16": 8e-4}


class Sharing(u.Paged):
    """seqs = [(new tokens, own positions with them)], behind `shared` pages that are the same for all."""

    def __init__(self, pkg, seed, seqs, heads, d, page, dtype, cache, shared, **more):
        gap = more.pop("gap", 0)
        super().__init__(pkg, seed, list(seqs) + [(0, shared * page)], heads, d, page, dtype, cache, **more)
        own, self.shared = self.table[:-1], shared
        self.prefix = self.table[-1, :shared].clone()
        need = max([-(-n // page) for _, n in seqs] + [0]) + more.get("slack", 0)
        self.table = torch.cat((self.prefix.expand(len(seqs), shared), own[:, :need]), 1).contiguous()
        self.pitch = shared + need
        self.seqs = [(new, shared * page + n) for new, n in seqs]
        self.starts_h, self.starts, self.lens = self.starts_h[:-1], self.starts[:-1].contiguous(), self.lens[:-1] + shared * page
        self.tokens = self.starts_h[-1] + gap


def run(pkg, dev, cache, q, o=None):
    o = torch.full_like(q, 55.0) if o is None else o
    # a row's own entries for the prefix are not looked at
    table = cache.table
    cache.table = table.clone()
    cache.table[:, :cache.shared] = -3
    try:
        dev.attention_paged_prefix(cache.view(), cache.batch(), u.codes(pkg.capi)[cache.dtype], q.shape[1], cache.shared * cache.page, u.ptr(cache.prefix), u.ptr(q), u.ptr(o),
                                   stream=u.stream())
        torch.cuda.synchronize()
    finally:
        cache.table = table
    assert dev.status() == 0
    return o


def check(cache, q, o, scale=1.0):
    used = cache.starts_h[-1]
    assert (o[used:] == 55).all()
    want, got = cache.attend(q)[:used], o[:used].double()
    assert torch.isfinite(got).all()
    for b in range(len(cache.seqs)):
        at = slice(cache.starts_h[b], cache.starts_h[b + 1])
        if at.start == at.stop:
            continue
        off = (got[at] - want[at]).norm() / want[at].norm()
        assert off <= REL[cache.dtype], (b, cache.seqs[b], float(off))
        worst = ((got[at] - want[at]).abs().amax(-1) / want[at].square().mean(-1).sqrt()).max()
        assert worst <= 12 * REL[cache.dtype], (b, cache.seqs[b], float(worst))


def one(pkg, dev, seed, seqs, hq, hkv, d, page, dtype, held, shared, **more):
    cache = Sharing(pkg, seed, seqs, hkv, d, page, dtype, held, shared, **more)
    q = u.normal(u.gen(seed + 1), (cache.tokens, hq, d), 1.5).to(u.TORCH[dtype])
    check(cache, q, run(pkg, dev, cache, q))


TYPES = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "i8"), ("f16", "i8")]


@pytest.mark.parametrize("dtype,held", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (1, 1), (14, 2), (20, 1)])
@pytest.mark.parametrize("shared", [1, 40])
def test_single_tokens(dev, pkg, dtype, held, d, hq, hkv, shared):
    one(pkg, dev, 11, [(1, n) for n in (1, 2, 15, 16, 17, 31, 64, 65, 129, 700, 1500)], hq, hkv, d, 16, dtype, held, shared)


@pytest.mark.parametrize("dtype,held", TYPES)
@pytest.mark.parametrize("batch", [1, 2, 3])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2)])
def test_few_rows(dev, pkg, dtype, held, batch, hq, hkv):
    """As many rows as one tile of the kernel for few has, and fewer."""
    one(pkg, dev, 12, [(1, 20 + 60 * b) for b in range(batch)], hq, hkv, 128, 16, dtype, held, 33)


@pytest.mark.parametrize("dtype,held", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (14, 2)])
def test_mixed(dev, pkg, dtype, held, d, hq, hkv):
    """Chunks, proposed tokens and single ones, sequences without new tokens, rows behind the last sequence."""
    one(pkg, dev, 13, [(1, 300), (0, 77), (130, 130), (3, 500), (57, 400), (0, 1), (1, 1), (64, 128), (31, 900)], hq, hkv, d, 32, dtype, held, 9, slack=2, gap=5)


@pytest.mark.parametrize("page,shared", [(1, 37), (3, 50), (8, 5), (24, 7), (64, 3), (96, 2), (128, 1), (1000, 1)])
@pytest.mark.parametrize("held", ["bf16", "i8"])
@pytest.mark.parametrize("new", [1, 6])
def test_page_sizes(dev, pkg, page, shared, held, new):
    one(pkg, dev, 14, [(new, 515), (1, 44), (new, 12), (1, page), (1, page + 1), (new, 325)], 8, 2, 128, page, "bf16", held, shared)


@pytest.mark.parametrize("held", ["bf16", "i8"])
@pytest.mark.parametrize("batch", [3, 40])
def test_long(dev, pkg, held, batch):
    """Every sequence has pages of its own below the prefix as well, so the batch is held small."""
    one(pkg, dev, 15, [(1, 1 + 29 * i % 97) for i in range(batch)], 8, 2, 64 if held == "i8" else 128, 64, "bf16", held, 200)


@pytest.mark.parametrize("dtype,held", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 24, 128])
def test_prefix_of_many_rows(dev, pkg, dtype, held, d, page):
    """The prefix on tcgen05 in blocks of 256 rows, the last ones in part, its end inside a tile; single tokens, some, and a chunk behind it."""
    one(pkg, dev, 26, [(1, 1 + 29 * i % 97) for i in range(60)] + [(7, 50), (100, 130), (1, 700)], 28, 4, d, page, dtype, held, 7800 // page)


@pytest.mark.parametrize("held", ["bf16", "i8"])
def test_prefix_of_one_tile_and_many_rows(dev, pkg, held):
    """So many rows that even a short prefix is tcgen05's, and blocks are whole."""
    one(pkg, dev, 27, [(20, 60)] * 80, 32, 2, 128, 64, "bf16", held, 2)


@pytest.mark.parametrize("page", [3, 20])
def test_many_rows_on_pages_that_boxes_do_not_fit(dev, pkg, page):
    one(pkg, dev, 28, [(1, 30)] * 50 + [(30, 60)], 16, 2, 64, page, "f16", "f16", 1500 // page)


@pytest.mark.parametrize("batch", [150, 600])
@pytest.mark.parametrize("held", ["f16", "i8"])
def test_many_sequences(dev, pkg, batch, held):
    one(pkg, dev, 16, [(1, 1 + 37 * i % 211) for i in range(batch)], 8, 4, 128, 16, "f16", held, 3)


def test_the_same_as_attention_over_pages(dev, pkg):
    for held in ("bf16", "i8"):
        cache = Sharing(pkg, 17, [(1, 100), (5, 60), (1, 7)], 2, 128, 16, "bf16", held, 30)
        q = u.normal(u.gen(18), (cache.tokens, 16, 128)).bfloat16()
        plain = torch.empty_like(q)
        dev.attention_paged(cache.view(), cache.batch(), pkg.capi.BF16, 16, u.ptr(q), u.ptr(plain), stream=u.stream())
        o = run(pkg, dev, cache, q)
        assert (o.double() - plain.double()).norm() <= 2 * REL["bf16"] * plain.double().norm()


def test_without_a_prefix(dev, pkg):
    cache = Sharing(pkg, 19, [(1, 100), (5, 60)], 2, 64, 16, "bf16", "bf16", 0)
    q = u.normal(u.gen(18), (cache.tokens, 4, 64)).bfloat16()
    plain = torch.empty_like(q)
    dev.attention_paged(cache.view(), cache.batch(), pkg.capi.BF16, 4, u.ptr(q), u.ptr(plain), stream=u.stream())
    assert torch.equal(run(pkg, dev, cache, q), plain)


@pytest.mark.parametrize("held", ["bf16", "i8"])
@pytest.mark.parametrize("new,batch", [(1, 2), (1, 30), (20, 3)])
def test_all_weight_on_one_side(dev, pkg, held, new, batch):
    """Scores that leave one of the two parts nothing: what is left is the other's, and its V where one key takes all."""
    for part in (0, 1):
        cache = Sharing(pkg, 20, [(new, 40)] * batch, 1, 64, 16, "bf16", held, 4)
        for b in range(batch):
            for i in range(cache.pitch):
                k = cache.kv[0][int(cache.table[b, i])]
                first = i < 4
                k[..., 0] = 100 if first == (part == 0) else -100
                if held == "i8":
                    cache.scales[0][int(cache.table[b, i])] = 1.0
        q = u.normal(u.gen(21), (cache.tokens, 2, 64)).bfloat16()
        q[..., 0] = 300.0
        o = run(pkg, dev, cache, q)
        check(cache, q, o)


def test_parts_whose_scores_are_all_minus_infinity(dev, pkg):
    """They weigh nothing beside the other part; both: NaN, as of one softmax over all of them."""
    for spoilt in ((True, False), (False, True), (True, True)):
        for new, batch in ((1, 2), (1, 30), (20, 3)):
            cache = Sharing(pkg, 22, [(new, 40)] * batch, 1, 64, 16, "bf16", "bf16", 4, junk=0.0)
            for b in range(batch):
                for i in range(cache.pitch):
                    if spoilt[0 if i < 4 else 1]:
                        cache.kv[0][int(cache.table[b, i])][..., 0] = -float("inf")
            q = u.normal(u.gen(21), (cache.tokens, 2, 64)).abs().bfloat16() + 0.5
            o = torch.empty_like(q)
            o = run(pkg, dev, cache, q)
            if all(spoilt):
                assert torch.isnan(o).all()
            else:
                assert torch.isfinite(o).all()
                check(cache, q, o)


def test_not_finite_scores_and_values(dev, pkg):
    """A NaN or +inf score, in either part, makes NaN of the rows that see it and of no others."""
    for where in (1, 4 * 16 + 3):
        for bad in (float("nan"), float("inf")):
            for new, batch in ((1, 3), (1, 30)):
                cache = Sharing(pkg, 23, [(new, 40)] * batch, 1, 64, 16, "bf16", "bf16", 4, junk=0.0)
                cache.kv[0][int(cache.table[1, where // 16]), 0, where % 16, 0] = bad
                q = u.normal(u.gen(21), (cache.tokens, 2, 64)).abs().bfloat16() + 0.5
                o = run(pkg, dev, cache, q)
                gone = torch.isnan(o).all(-1).all(-1)
                if where < 64:
                    assert gone.all()
                else:
                    assert gone.tolist() == [b == 1 for b in range(batch)] and torch.isfinite(o[~gone]).all()


def test_results_do_not_depend_on_the_run_or_the_stream(dev, pkg):
    cache = Sharing(pkg, 24, [(1, 1500), (20, 300), (1, 20)] * 4, 4, 128, 16, "bf16", "i8", 100)
    q = u.normal(u.gen(22), (cache.tokens, 16, 128)).bfloat16()
    first = run(pkg, dev, cache, q)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(5):
            assert torch.equal(run(pkg, dev, cache, q), first)


@pytest.mark.parametrize("batch", [2, 20])
def test_in_a_graph(dev, pkg, batch):
    """Two graphs captured once, replayed in turn for other lengths and another prefix of the same length."""
    cache = Sharing(pkg, 25, [(1, 300)] * batch, 2, 128, 16, "bf16", "bf16", 12, junk=0.0)
    q = u.normal(u.gen(24), (batch, 8, 128)).bfloat16()
    outs = [run(pkg, dev, cache, q), torch.zeros_like(q)]
    view, step, graphs, s = cache.view(), cache.batch(), [], torch.cuda.Stream()
    for o in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            dev.attention_paged_prefix(view, step, pkg.capi.BF16, 8, 192, u.ptr(cache.prefix), u.ptr(q), u.ptr(o), stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    for turn in range(3):
        lens = [192 + 1 + (77 * b + 31 * turn) % 300 for b in range(batch)]
        cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        cache.seqs = [(1, n) for n in lens]
        cache.prefix.copy_(cache.prefix.flip(0))
        cache.table[:, :12] = cache.prefix
        for o in outs:
            o.zero_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert dev.status() == 0
        for o in outs:
            check(cache, q, o)


@pytest.mark.parametrize("held", ["bf16", "i8"])
def test_what_is_outside_is_reported(dev, pkg, held):
    """The other sequences are served all the same, and what is left out is not written."""
    def page(c):
        c.table[1, c.shared] = c.pages + 5

    def length(c):
        c.lens[1] = c.pitch * c.page + 1

    def short(c):
        c.lens[1] = c.shared * c.page + c.seqs[1][0] - 1

    def inside(c):
        c.lens[1] = c.seqs[1][0]

    def order(c):  # tokens behind starts[batch], which no row of the prefix stands for
        c.starts[3] = c.starts_h[1]

    for spoil in (page, length, short, inside, order):
        for news in ((1, 1, 1), (4, 4, 4), (30, 4, 40)):
            c = Sharing(pkg, 3, [(news[0], 80), (news[1], 60), (news[2], 70)], 2, 64, 16, "bf16", held, 3)
            spoil(c)
            q = u.normal(u.gen(4), (c.tokens, 4, 64)).bfloat16()
            o = torch.full_like(q, 55.0)
            dev.attention_paged_prefix(c.view(), c.batch(), pkg.capi.BF16, 4, 48, u.ptr(c.prefix), u.ptr(q), u.ptr(o), stream=u.stream())
            with pytest.raises(pkg.hal.KernelError, match="left it out"):
                pkg.hal.check(pkg.capi.lib().tsm100_stream_synchronize(dev._h, None))
            if spoil is not page:
                assert (o[c.starts_h[1]:c.starts_h[2]] == 55).all()
            if spoil is order:
                assert (o[c.starts_h[2]:] == 55).all()
            c.seqs = [c.seqs[0], (0, 0), c.seqs[2]]
            want = c.attend(q)
            for b in (0, 2) if spoil is not order else (0,):
                at = slice(c.starts_h[b], c.starts_h[b + 1])
                assert (o[at].double() - want[at]).norm() <= REL["bf16"] * want[at].norm(), (spoil.__name__, news, b)
            assert dev.status() == 0


@pytest.mark.parametrize("held", ["bf16", "i8"])
@pytest.mark.parametrize("news,group,page", [((1, 1, 1), 4, 16), ((3, 1, 0), 4, 16), ((3, 40, 9), 4, 16), ((3, 40, 9), 5, 3)])
def test_any_number_of_new_tokens_allowed(dev, pkg, news, group, page, held):
    """max_new as large as it goes takes no memory by itself: the same result, bit for bit, as with the call's tokens."""
    cache = Sharing(pkg, 31, list(zip(news, (90, 700, 33))), 2, 64, page, "bf16", held, 7)
    q = u.normal(u.gen(32), (cache.tokens, 2 * group, 64)).bfloat16()
    got = []
    for most in (cache.tokens, 2**31 - 1):
        batch = pkg.hal.PagedBatch(3, cache.tokens, most, 0, cache.pitch, u.ptr(cache.table), u.ptr(cache.lens), u.ptr(cache.starts))
        o = torch.full_like(q, 55.0)
        dev.attention_paged_prefix(cache.view(), batch, pkg.capi.BF16, 2 * group, cache.shared * cache.page, u.ptr(cache.prefix), u.ptr(q), u.ptr(o), stream=u.stream())
        torch.cuda.synchronize()
        assert dev.status() == 0
        got.append(o)
    assert torch.equal(*got)
    check(cache, q, got[0])


def test_refusals(dev, pkg):
    capi, hal = pkg.capi, pkg.hal
    x = torch.zeros(4096, device=u.GPU)
    p = x.data_ptr()

    def bad(match, dtype=capi.BF16, heads_q=4, cache=None, q=p, o=p, prefix_len=16, prefix=p):
        kv = dict(dtype=capi.BF16, heads_kv=2, head_dim=64, page_size=16, pages=2, k=p, v=p) | (cache or {})
        with pytest.raises(hal.KernelError, match="attention_paged_prefix: .*" + match):
            dev.attention_paged_prefix(hal.PagedKv(**kv), hal.PagedBatch(1, 1, 1, 0, 4, p, p, p), dtype, heads_q, prefix_len, prefix, q, o, stream=u.stream())

    bad("dtype must be", dtype=capi.F32)
    bad("must hold", cache={"dtype": capi.F16})
    bad("head_dim must be 64 or 128", cache={"head_dim": 96})
    bad("multiple of heads_kv", heads_q=3)
    bad("null buffer", q=0)
    bad("16-byte aligned", o=p + 2)
    bad("multiple of page_size", prefix_len=8)
    bad("multiple of page_size", prefix_len=-16)
    bad("more than a row", prefix_len=80)
    bad("null prefix", prefix=0)
    bad("prefix does not start", prefix=p + 2)
    dev.attention_paged_prefix(hal.PagedKv(capi.BF16, 2, 64, 16, 2, p, p), hal.PagedBatch(0, 0, 0, 0, 1, 0, 0, 0), capi.BF16, 4, 16, 0, 0, 0, stream=u.stream())
