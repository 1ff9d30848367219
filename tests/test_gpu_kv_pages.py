"""The paged KV cache: what is appended lies where the table says, number by number, and is read back; nothing else is touched."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu
# sequences without tokens, of one token, whose tokens begin and end inside pages, and fill them exactly
MIXES = [[(1, 1)], [(1, 40), (1, 16), (1, 17)], [(0, 33), (5, 5), (0, 0), (70, 133), (16, 32)], [(200, 1000), (1, 999), (64, 64)], [(0, 4)]]


def append(pkg, dev, cache, k, v):
    dev.kv_page_append(cache.view(), cache.batch(), u.codes(pkg.capi)[cache.dtype], u.ptr(k), u.ptr(v), stream=u.stream())


@pytest.mark.parametrize("seqs", MIXES)
@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("heads,d,dtype,held", [(8, 128, "bf16", "bf16"), (2, 64, "f16", "i8"), (3, 128, "bf16", "i8"), (1, 16, "f16", "f16"), (5, 240, "f16", "i8"),
                                                (2, 256, "bf16", "i8")])
def test_append_and_read(dev, pkg, seqs, page, heads, d, dtype, held):
    cache = u.Paged(pkg, 5, seqs, heads, d, page, dtype, held, slack=1, gap=3)
    g, t = u.gen(6), u.TORCH[dtype]
    new = [u.normal(g, (cache.tokens, heads, d)).to(t) for _ in range(2)]
    if cache.tokens > 4:
        new[0][2] = 0  # a token of zeros: step 0
    want, steps = [x.clone() for x in cache.kv], [None if x is None else x.clone() for x in cache.scales]
    for w in range(2):
        q, s = u.quantise(new[w].float()) if held == "i8" else (new[w], None)
        for b, (count, n) in enumerate(seqs):
            for i in range(count):
                pos, token = n - count + i, cache.starts_h[b] + i
                page_id = int(cache.table[b, pos // page])
                want[w][page_id, :, pos % page] = q[token]
                if s is not None:
                    steps[w][page_id, :, pos % page] = s[token]
    append(pkg, dev, cache, *new)
    for w in range(2):
        a, b = cache.kv[w], want[w]
        assert torch.equal(a.view(torch.int16), b.view(torch.int16)) if held != "i8" else torch.equal(a, b)
        if held == "i8":
            assert torch.equal(cache.scales[w].view(torch.int32), steps[w].view(torch.int32))
    total = cache.places_h[-1]
    out = [torch.full((total + 1, heads, d), 77.0, dtype=t, device=u.GPU) for _ in range(2)]
    dev.kv_page_read(cache.view(), cache.batch(whole=True), u.codes(pkg.capi)[dtype], u.ptr(out[0]), u.ptr(out[1]), stream=u.stream())
    for w in range(2):
        assert (out[w][total:] == 77).all()
        for b in range(len(seqs)):
            got = out[w][cache.places_h[b]:cache.places_h[b + 1]]
            assert torch.equal(got, cache.rows(w, b).float().to(t)), (w, b)  # the product in f32, rounded to the type
    assert dev.status() == 0


def test_reading_the_new_tokens_only(dev, pkg):
    cache = u.Paged(pkg, 9, [(3, 50), (20, 20)], 4, 128, 16, "bf16", "bf16")
    out = [torch.zeros((cache.tokens, 4, 128), dtype=torch.bfloat16, device=u.GPU) for _ in range(2)]
    dev.kv_page_read(cache.view(), cache.batch(), pkg.capi.BF16, u.ptr(out[0]), u.ptr(out[1]), stream=u.stream())
    for w in range(2):
        assert torch.equal(out[w][:3], cache.rows(w, 0)[47:].bfloat16()) and torch.equal(out[w][3:], cache.rows(w, 1).bfloat16())


@pytest.mark.parametrize("held", ["bf16", "i8"])
def test_what_is_outside_is_left_out_and_reported(dev, pkg, held):
    """A page that does not exist, a sequence longer than its row of the table, more tokens than positions, than max_new, than the call has: the other
    sequences are served."""
    def fresh():
        return u.Paged(pkg, 3, [(4, 40), (4, 30), (4, 20)], 2, 64, 16, "bf16", held)

    def page(c):
        c.table[1, 1] = c.pages

    def negative(c):
        c.table[1, 1] = -1

    def length(c):
        c.lens[1] = c.pitch * c.page + 1

    def short(c):
        c.lens[1] = 3

    def backwards(c):
        c.starts[1], c.starts[2] = 9, 8  # -1 tokens

    for spoil in (page, negative, length, short, backwards):
        c = fresh()
        before = [x.clone() for x in c.kv]
        spoil(c)
        k = torch.full((c.tokens, 2, 64), 3.0, dtype=torch.bfloat16, device=u.GPU)
        append(pkg, dev, c, k, k)
        with pytest.raises(pkg.hal.KernelError, match="left it out"):
            pkg.hal.check(pkg.capi.lib().tsm100_stream_synchronize(dev._h, None))
        for w in range(2):
            here = before[w].clone()
            here[int(c.table[2, 1]), :, 0:4] = 127 if held == "i8" else 3.0
            here[int(c.table[0, 2]), :, 4:8] = 127 if held == "i8" else 3.0
            if spoil is not backwards:  # the order of such starts says nothing about who has which token
                assert torch.equal(c.kv[w].nan_to_num(5.0) if held != "i8" else c.kv[w], here.nan_to_num(5.0) if held != "i8" else here), spoil.__name__
        assert dev.status() == 0


def test_refusals(dev, pkg):
    capi, hal = pkg.capi, pkg.hal
    x = torch.zeros(4096, device=u.GPU)
    p = x.data_ptr()

    def bad(match, dtype=capi.BF16, cache=None, batch=None, k=p, v=p):
        kv = dict(dtype=capi.BF16, heads_kv=2, head_dim=64, page_size=16, pages=2, k=p, v=p, k_scales=0, v_scales=0) | (cache or {})
        b = dict(batch=1, tokens=1, max_new=1, max_len=0, table_pitch=1, table=p, lens=p, starts=p) | (batch or {})
        for call in (dev.kv_page_append, dev.kv_page_read):
            with pytest.raises(hal.KernelError, match=match):
                call(hal.PagedKv(**kv), hal.PagedBatch(**b), dtype, k, v, stream=u.stream())

    bad("dtype must be", dtype=capi.F32)
    bad("must hold", cache={"dtype": capi.F16})
    bad("bad cache shape", cache={"heads_kv": 0})
    bad("bad cache shape", cache={"page_size": 0})
    bad("bad cache shape", cache={"page_size": 5000})
    bad("bad cache shape", cache={"pages": -1})
    bad("head_dim", cache={"head_dim": 72})
    bad("head_dim", cache={"head_dim": 272})
    bad("too many pages", cache={"pages": 1 << 30, "heads_kv": 2})
    bad("bad batch shape", batch={"tokens": -1})
    bad("too many positions", batch={"table_pitch": 1 << 28})
    bad("null table", batch={"table": 0})
    bad("null table", batch={"lens": 0})
    bad("null table", batch={"starts": 0})
    bad("null cache", cache={"k": 0})
    bad("cache must be 16-byte", cache={"v": p + 2})
    bad("needs scales", cache={"dtype": capi.I8})
    bad("null buffer", k=0)
    bad("16-byte aligned", v=p + 2)
    # nothing to do
    dev.kv_page_append(hal.PagedKv(capi.BF16, 2, 64, 16, 2, p, p), hal.PagedBatch(0, 0, 0, 0, 0, 0, 0, 0), capi.BF16, 0, 0, stream=u.stream())
