"""One layer of a decoder with an encoder, served to many sequences that begin with the same prompt: 8-bit weights and activations, the prompt's keys and values held and read
once, cross attention to each sequence's encoder states.

    residual norm (8-bit rows) -> Q, K, V products -> rotary embedding -> append to the pages -> attention on the shared prompt and a sequence's own tokens ->
    rows in 8 bits -> output product -> residual norm -> Q product -> cross attention over the encoder's pages -> rows in 8 bits -> output product ->
    residual norm -> gate and up in one product -> SiLU * up as rows in 8 bits -> down product

    python examples/shared_prompt_layer.py
"""
from __future__ import annotations

import sys
import time
from dataclasses import dataclass
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import __graft_entry__ as entry  # noqa: E402

pkg = entry.load_package()
capi, hal = pkg.capi, pkg.hal


@dataclass
class Config:
    hidden: int = 1024
    inner: int = 2816
    heads_q: int = 16
    heads_kv: int = 4
    head_dim: int = 64
    page: int = 16
    theta: float = 10000.0
    eps: float = 1e-5


class Weights8:
    """[n, k] weights as whole numbers with a step for every output."""

    def __init__(self, w: torch.Tensor):
        self.n, self.k = w.shape
        self.steps = w.float().abs().amax(1) / 127
        self.numbers = torch.round(w.float() / self.steps[:, None]).to(torch.int8)

    def dense(self) -> torch.Tensor:
        return self.numbers.double() * self.steps.double()[:, None]


class Cache:
    """Pages of keys and values in bf16, handed out as sequences grow."""

    def __init__(self, c: Config, pages: int):
        self.c, self.free = c, list(range(pages))[::-1]
        self.k, self.v = (torch.zeros((pages, c.heads_kv, c.page, c.head_dim), dtype=torch.bfloat16, device="cuda:0") for _ in range(2))
        self.view = hal.PagedKv(capi.BF16, c.heads_kv, c.head_dim, c.page, pages, self.k.data_ptr(), self.v.data_ptr())

    def grow(self, held: list, length: int) -> None:
        while len(held) * self.c.page < length:
            held.append(self.free.pop())


def on_device(x: list) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int32).to("cuda:0")


class Step:
    """The sequences of a call: news[b] new tokens of lens[b] positions on pages[b], and the arrays that the kernels read."""

    def __init__(self, news: list, lens: list, pages: list):
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        wide = max(1, max(len(p) for p in pages))
        self.news, self.lens, self.tokens = news, lens, starts[-1]
        self.table, self.lens_d, self.starts = on_device([p + [0] * (wide - len(p)) for p in pages]), on_device(lens), on_device(starts)
        self.batch = hal.PagedBatch(len(news), self.tokens, max(news), 0, wide, self.table.data_ptr(), self.lens_d.data_ptr(), self.starts.data_ptr())


class Layer:
    def __init__(self, dev: "hal.CudaSm100Device", c: Config, seed: int = 0):
        self.dev, self.c = dev, c
        g = torch.Generator(device="cuda:0")
        g.manual_seed(seed)

        def weights(n, k):
            return Weights8(torch.randn((n, k), generator=g, device="cuda:0") * k ** -0.5)

        q, kv = c.heads_q * c.head_dim, c.heads_kv * c.head_dim
        self.wq, self.wk, self.wv, self.wo = weights(q, c.hidden), weights(kv, c.hidden), weights(kv, c.hidden), weights(c.hidden, q)
        self.cross_q, self.cross_k, self.cross_v, self.cross_o = weights(q, c.hidden), weights(kv, c.hidden), weights(kv, c.hidden), weights(c.hidden, q)
        self.gate_up, self.down = weights(2 * c.inner, c.hidden), weights(c.hidden, c.inner)
        self.norms = [(1 + 0.1 * torch.randn(c.hidden, generator=g, device="cuda:0")).bfloat16() for _ in range(3)]

    def _norm(self, x, residual, weight, st):
        """(x + residual, its norm as whole numbers, their steps)"""
        total, numbers, steps = torch.empty_like(x), torch.empty_like(x, dtype=torch.int8), torch.empty(x.shape[0], device=x.device)
        self.dev.add_rms_norm(capi.BF16, x.shape[0], self.c.hidden, self.c.eps, x.data_ptr(), 0 if residual is None else residual.data_ptr(), total.data_ptr(),
                              weight.data_ptr(), numbers.data_ptr(), out_dtype=capi.I8, scales=steps.data_ptr(), stream=st)
        return total, numbers, steps

    def _rows(self, x, cols, st, gated=False):
        """The rows of x, or of silu(gate) * up where it has both, as whole numbers and steps."""
        numbers, steps = torch.empty((x.shape[0], cols), dtype=torch.int8, device=x.device), torch.empty(x.shape[0], device=x.device)
        self.dev.quantise_rows(capi.BF16, x.shape[0], cols, x.data_ptr(), numbers.data_ptr(), steps.data_ptr(),
                               up=x[:, cols:].data_ptr() if gated else 0, pitch=x.shape[1], stream=st)
        return numbers, steps

    def _product(self, numbers, steps, w, st):
        out = torch.empty((numbers.shape[0], w.n), dtype=torch.bfloat16, device=numbers.device)
        self.dev.gemm_i8(capi.BF16, numbers.shape[0], w.n, w.k, numbers.data_ptr(), steps.data_ptr(), w.numbers.data_ptr(), w.steps.data_ptr(), out.data_ptr(), stream=st)
        return out

    def encode(self, states: torch.Tensor, cache: Cache, step: Step) -> None:
        """Keys and values of the encoder's states [positions, hidden] of all sequences, into its pages."""
        st = torch.cuda.current_stream().cuda_stream
        numbers, steps = self._rows(states, self.c.hidden, st)
        k, v = self._product(numbers, steps, self.cross_k, st), self._product(numbers, steps, self.cross_v, st)
        self.dev.kv_page_append(cache.view, step.batch, capi.BF16, k.data_ptr(), v.data_ptr(), stream=st)

    def step(self, x: torch.Tensor, cache: Cache, step: Step, shared: torch.Tensor, encoded: Cache, encoder: Step) -> torch.Tensor:
        """x [tokens, hidden] bf16: the new tokens of all sequences, behind the pages `shared` that they begin with; `encoder`: their encoders' positions, with the same
        new tokens."""
        c, dev, st = self.c, self.dev, torch.cuda.current_stream().cuda_stream
        width = c.heads_q * c.head_dim
        h, numbers, steps = self._norm(x, None, self.norms[0], st)
        q, k, v = (self._product(numbers, steps, w, st) for w in (self.wq, self.wk, self.wv))
        at = 0
        for new, n in zip(step.news, step.lens):  # every sequence is at a position of its own
            for t, heads in ((q, c.heads_q), (k, c.heads_kv)):
                if new:
                    dev.rope(capi.BF16, 1, new, heads, c.head_dim, n - new, c.theta, t[at:].data_ptr(), stream=st)
            at += new
        dev.kv_page_append(cache.view, step.batch, capi.BF16, k.data_ptr(), v.data_ptr(), stream=st)
        o = torch.empty_like(q)
        dev.attention_paged_prefix(cache.view, step.batch, capi.BF16, c.heads_q, shared.numel() * c.page, shared.data_ptr(), q.data_ptr(), o.data_ptr(), stream=st)
        h, numbers, steps = self._norm(self._product(*self._rows(o, width, st), self.wo, st), h, self.norms[1], st)
        q = self._product(numbers, steps, self.cross_q, st)
        dev.attention_paged_cross(encoded.view, encoder.batch, capi.BF16, c.heads_q, q.data_ptr(), o.data_ptr(), stream=st)
        h, numbers, steps = self._norm(self._product(*self._rows(o, width, st), self.cross_o, st), h, self.norms[2], st)
        both = self._product(numbers, steps, self.gate_up, st)
        return self._product(*self._rows(both, c.inner, st, gated=True), self.down, st) + h


def serve(layer: Layer, prompt: torch.Tensor, states: list, first: list, generated: int):
    """The prompt once, then for each sequence its first own tokens and what the layer gives back, all behind the prompt's whole pages.  states[b]: [positions, hidden] of
    an encoder (any number, none too).  Yields (step, input, output); the prompt's own step first."""
    c, batch = layer.c, len(states)
    most = prompt.shape[0] + max(f.shape[0] for f in first) + generated
    cache = Cache(c, -(-most // c.page) * (batch + 1))
    encoded = Cache(c, sum(-(-s.shape[0] // c.page) for s in states) + 1)
    enc_lens, enc_pages = [s.shape[0] for s in states], [[] for _ in states]
    for held, n in zip(enc_pages, enc_lens):
        encoded.grow(held, n)
    layer.encode(torch.cat(states), encoded, Step(enc_lens, enc_lens, enc_pages))
    # the prompt: one sequence, nothing before it; it has no encoder
    held = []
    cache.grow(held, prompt.shape[0])
    step = Step([prompt.shape[0]], [prompt.shape[0]], [held])
    none = torch.zeros(0, dtype=torch.int32, device="cuda:0")
    yield step, prompt, layer.step(prompt, cache, step, none, encoded, Step([prompt.shape[0]], [0], [[]]))
    # whole pages of it are shared; what is left over every sequence repeats as tokens of its own
    whole = prompt.shape[0] // c.page
    shared, pages, done = on_device(held[:whole]), [held[:whole] for _ in states], [whole * c.page] * batch
    x = [torch.cat((prompt[whole * c.page:], f)) for f in first]
    for _ in range(1 + generated):
        news = [t.shape[0] for t in x]
        done = [n + new for n, new in zip(done, news)]
        for p, n in zip(pages, done):
            cache.grow(p, n)
        step, tokens = Step(news, list(done), pages), torch.cat(x)
        y = layer.step(tokens, cache, step, shared, encoded, Step(news, enc_lens, enc_pages))
        yield step, tokens, y
        at = 0
        for b, new in enumerate(news):
            at += new
            x[b] = torch.nn.functional.normalize(y[at - 1:at].float(), dim=-1).mul(c.hidden ** 0.5).bfloat16()


def main() -> None:
    c = Config()
    dev = hal.CudaSm100Device(0)
    layer = Layer(dev, c)
    prompt, generated = torch.randn((4000, c.hidden), device="cuda:0").bfloat16(), 32
    states = [torch.randn((100 + 37 * b % 400, c.hidden), device="cuda:0").bfloat16() for b in range(48)]
    first = [torch.randn((1 + b % 5, c.hidden), device="cuda:0").bfloat16() for b in range(48)]
    for _ in serve(layer, prompt, states, first, 2):
        pass
    torch.cuda.synchronize()
    began, tokens, steps = time.perf_counter(), 0, 0
    for step, _, _ in serve(layer, prompt, states, first, generated):
        tokens, steps = tokens + step.tokens, steps + 1
    torch.cuda.synchronize()
    assert dev.status() == 0
    took = time.perf_counter() - began
    print(f"{steps} steps, {tokens} tokens of {len(states)} sequences behind a prompt of {prompt.shape[0]} (8-bit weights): {1e3 * took / steps:.2f} ms a step")


if __name__ == "__main__":
    main()
