"""Plain 64-bit restatements of the serving operators, and paged caches to test them on."""
import torch

GPU = "cuda:0"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# half a unit in the last place of 1.0: one rounding to the type, relative (24, 8 and 11 significant bits)
HALF_ULP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
SMALLEST = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}


def codes(capi):
    return {"f32": capi.F32, "bf16": capi.BF16, "f16": capi.F16, "i8": capi.I8}


def gen(seed):
    g = torch.Generator(device=GPU)
    g.manual_seed(seed)
    return g


def normal(g, shape, sigma=1.0):
    return torch.randn(shape, generator=g, device=GPU) * sigma


def ptr(t):
    return 0 if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def quantise(x):
    """Rows of f32 x as whole numbers and steps, by the definition's own f32 operations: one multiplication, one division, to nearest even."""
    step = x.abs().amax(-1, keepdim=True) * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=x.device)
    return torch.round(torch.where(step > 0, x / step, torch.zeros_like(x))).to(torch.int8), step.squeeze(-1)


class Paged:
    """A paged cache of `seqs` = [(new tokens, positions with them)], pages in random order, whatever no sequence has filled with `junk`."""

    def __init__(self, pkg, seed, seqs, heads, d, page, dtype, cache, junk=float("nan"), spare=2, slack=0, gap=0):
        self.pkg, self.capi = pkg, pkg.capi
        self.seqs, self.heads, self.d, self.page, self.dtype, self.cache = seqs, heads, d, page, dtype, cache
        g = gen(seed)
        need = [-(-n // page) for _, n in seqs]
        self.pages, self.pitch = sum(need) + spare, max(need + [0]) + slack
        order, at = torch.randperm(self.pages, generator=g, device=GPU).int(), 0
        self.table = torch.full((len(seqs), max(self.pitch, 1)), -7, dtype=torch.int32, device=GPU)  # entries behind a sequence's end are never looked at
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.starts_h = [0]
        for new, _ in seqs:
            self.starts_h.append(self.starts_h[-1] + new)
        self.places_h = [0]
        for _, n in seqs:
            self.places_h.append(self.places_h[-1] + n)
        self.tokens = self.starts_h[-1] + gap
        self.lens, self.starts, self.places = (torch.tensor(x, dtype=torch.int32, device=GPU) for x in ([n for _, n in seqs], self.starts_h, self.places_h))
        shape = (self.pages, heads, page, d)
        self.kv, self.scales = [], []
        for _ in range(2):
            x = normal(g, shape) * torch.exp(normal(g, shape[:3] + (1,), 0.5))
            if cache == "i8":
                q, s = quantise(x)
            else:
                q, s = x.to(TORCH[cache]), None
            for_junk = torch.ones(shape[:3], dtype=torch.bool, device=GPU)
            for b, (_, n) in enumerate(seqs):
                for i in range(-(-n // page)):
                    for_junk[int(self.table[b, i]), :, :n - i * page] = False
            if cache == "i8":
                q[for_junk] = -128
                s[for_junk] = junk
            else:
                q[for_junk] = junk
            self.kv.append(q)
            self.scales.append(s)

    def view(self):
        return self.pkg.hal.PagedKv(codes(self.capi)[self.cache], self.heads, self.d, self.page, self.pages, ptr(self.kv[0]), ptr(self.kv[1]),
                                    ptr(self.scales[0]), ptr(self.scales[1]))

    def batch(self, whole=False, max_len=0):
        """The sequences' new tokens, or all their positions."""
        starts = self.places if whole else self.starts
        most = max([n if whole else new for new, n in self.seqs] + [0])
        tokens = self.places_h[-1] if whole else self.tokens
        return self.pkg.hal.PagedBatch(len(self.seqs), tokens, most, max_len, self.pitch, ptr(self.table), ptr(self.lens), ptr(starts))

    def rows(self, which, b):
        """[positions, heads, d] of sequence b in 64 bits."""
        n, out = self.seqs[b][1], []
        for i in range(-(-n // self.page)):
            page = int(self.table[b, i])
            x = self.kv[which][page].double()
            if self.scales[which] is not None:
                x = x * self.scales[which][page].double()[..., None]
            out.append(x.transpose(0, 1))
        return torch.cat(out)[:n] if out else torch.zeros((0, self.heads, self.d), dtype=torch.float64, device=GPU)

    def attend(self, q):
        """softmax(q k / sqrt d) v for q [tokens, heads_q, d], in 64 bits."""
        hq, out = q.shape[1], torch.zeros(q.shape, dtype=torch.float64, device=GPU)
        for b, (new, n) in enumerate(self.seqs):
            if new == 0:
                continue
            at = slice(self.starts_h[b], self.starts_h[b + 1])
            k, v = (self.rows(w, b).repeat_interleave(hq // self.heads, 1) for w in range(2))
            s = torch.einsum("qhd,khd->hqk", q[at].double(), k) / self.d ** 0.5
            hidden = torch.arange(n, device=GPU)[None] > torch.arange(n - new, n, device=GPU)[:, None]
            out[at] = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(hidden, -float("inf")), -1), v)
        return out
