"""Sequences as long as positions of 32 bits count, on one page that their tables repeat: served up to 2^31 - 4096 positions, left out beyond."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402

pytestmark = pytest.mark.gpu
MOST = 2**31 - 4096


class Repeated:
    """One KV head of 64 numbers in 8 bits, sequences = [(new tokens, positions)] all of whose positions lie in page 1 of 2."""

    def __init__(self, pkg, page, seqs):
        g = u.gen(7)
        self.pkg, self.page, self.seqs = pkg, page, seqs
        self.kv, self.scales = zip(*(u.quantise(u.normal(g, (2, 1, page, 64))) for _ in range(2)))
        self.pitch = (2**31 - 1) // page
        self.table = torch.ones((len(seqs), self.pitch), dtype=torch.int32, device=u.GPU)
        self.starts_h = [0]
        for new, _ in seqs:
            self.starts_h.append(self.starts_h[-1] + new)
        self.tokens = self.starts_h[-1]
        self.starts, self.lens = (torch.tensor(x, dtype=torch.int32, device=u.GPU) for x in (self.starts_h, [n for _, n in seqs]))
        self.q = u.normal(g, (self.tokens, 2, 64), 1.5).bfloat16()

    def call(self, dev, op):
        hal, capi = self.pkg.hal, self.pkg.capi
        kv = hal.PagedKv(capi.I8, 1, 64, self.page, 2, *map(u.ptr, self.kv), *map(u.ptr, self.scales))
        batch = hal.PagedBatch(len(self.seqs), self.tokens, max(new for new, _ in self.seqs), 0, self.pitch, u.ptr(self.table), u.ptr(self.lens), u.ptr(self.starts))
        o = torch.full_like(self.q, 55.0)
        if op == "prefix":
            dev.attention_paged_prefix(kv, batch, capi.BF16, 2, 16 * self.page, u.ptr(self.table), u.ptr(self.q), u.ptr(o), stream=u.stream())
        else:
            getattr(dev, op)(kv, batch, capi.BF16, 2, u.ptr(self.q), u.ptr(o), stream=u.stream())
        return o

    def want(self, b, causal):
        """Softmax over positions counted by their place in the page."""
        new, n = self.seqs[b]
        k, v = (x[1, 0].double() * s[1, 0].double()[:, None] for x, s in zip(self.kv, self.scales))
        place = torch.arange(self.page, device=u.GPU)
        out = []
        for r in range(new):
            sees = n - new + 1 + r if causal else n
            times = (sees - place + self.page - 1) // self.page  # positions with this place below `sees`
            s = self.q[self.starts_h[b] + r].double() @ k.T / 8
            p = torch.exp(s - s.amax(-1, keepdim=True)) * times
            out.append(p @ v / p.sum(-1, keepdim=True))
        return torch.stack(out)


# A row's largest number of the kernel's steps is 2^31 / (64 positions x 1184 warps or more), 28400: sums in f32 lose up to half a unit of 2^-24 of themselves a step,
# 2^-24 x 28400 / 2 = 8.5e-4 in all, the sum of weights and that of values each.  Beside the 6e-3 that attention over pages in bf16 is held to: 7.7e-3.
REL = 7.7e-3


@pytest.mark.parametrize("op", ["attention_paged", "attention_paged_cross", "prefix"])
def test_the_longest(dev, pkg, op):
    c = Repeated(pkg, 4096, [(1, MOST), (1, 70000)])
    o = c.call(dev, op)
    torch.cuda.synchronize()
    assert dev.status() == 0
    for b in range(2):
        want = c.want(b, op != "attention_paged_cross")
        assert (o[b].double() - want[0]).norm() <= REL * want.norm(), b


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("op", ["attention_paged", "attention_paged_cross", "prefix"])
def test_longer_ones_are_left_out(dev, pkg, op, new):
    c = Repeated(pkg, 127, [(new, 2**31 - 8), (new, 2500), (new, MOST + 1)])
    o = c.call(dev, op)
    with pytest.raises(pkg.hal.KernelError, match="left it out"):
        pkg.hal.check(pkg.capi.lib().tsm100_stream_synchronize(dev._h, None))
    assert (o[:new] == 55).all() and (o[2 * new:] == 55).all()
    want = c.want(1, op != "attention_paged_cross")
    assert (o[new:2 * new].double() - want).norm() <= 6e-3 * want.norm()
    assert dev.status() == 0
