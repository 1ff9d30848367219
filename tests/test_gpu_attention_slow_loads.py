"""16-bit attention on tcgen05, heads of 128, where loads are slower than products (few rows, many keys, every SM): a value tile is not used before it has landed, so that
repeated calls give the same bits, and the definition's result."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("news", [(5, 5, 5, 5), (5, 40, 6, 64)])
def test_over_pages(dev, pkg, news):
    cache = u.Paged(pkg, 5, [(new, 12000) for new in news], 8, 128, 64, "bf16", "bf16")
    q = u.normal(u.gen(6), (cache.tokens, 32, 128), 1.5).bfloat16()
    view, step, outs = cache.view(), cache.batch(), [torch.empty_like(q) for _ in range(3)]
    flush = torch.empty(64 << 20, dtype=torch.float32, device=u.GPU)
    for i in range(120):
        if i % 3 == 0:
            flush.fill_(i)  # the next call's loads come from memory
        dev.attention_paged(view, step, pkg.capi.BF16, 32, u.ptr(q), u.ptr(outs[min(i, 1) + (i > 60)]), stream=u.stream())
        if i > 0 and i % 20 == 0:
            assert torch.equal(outs[0], outs[1 + (i > 60)])
    assert dev.status() == 0
    at = slice(cache.starts_h[1], cache.starts_h[2])
    want = cache.attend(q)[at]
    assert (outs[0][at].double() - want).norm() <= 6e-3 * want.norm()


@pytest.mark.parametrize("seq_len", [19, 200])
def test_prefill(dev, pkg, seq_len):
    g, start, hq, hkv = u.gen(7), 15000, 32, 8
    q = u.normal(g, (seq_len, hq, 128)).bfloat16()
    k, v = (u.normal(g, (hkv, start + seq_len, 128)).bfloat16() for _ in range(2))
    first, again = torch.empty_like(q), torch.empty_like(q)
    flush = torch.empty(64 << 20, dtype=torch.float32, device=u.GPU)
    for i in range(60):
        if i % 3 == 0:
            flush.fill_(i)
        dev.attention_prefill(pkg.capi.BF16, hq, hkv, seq_len, start, start + seq_len, 128, u.ptr(q), u.ptr(k), u.ptr(v), u.ptr(again if i else first), stream=u.stream())
        if i and i % 15 == 0:
            assert torch.equal(first, again)
    assert dev.status() == 0
    s = torch.einsum("hd,kd->hk", q[-1, :4].double(), k[0].double()) / 128 ** 0.5
    want = torch.softmax(s, -1) @ v[0].double()
    assert (first[-1, :4].double() - want).norm() <= 6e-3 * want.norm()
