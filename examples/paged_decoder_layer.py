"""One decoder layer served the way the library's operators are meant to be used together: prompts in chunks and single tokens side by side, 4-bit
weights, a paged KV cache in 8 bits.

    residual norm (8-bit rows) -> Q, K, V products (4-bit weights) -> rotary embedding -> append to the pages -> attention over them ->
    output product -> residual norm (8-bit rows) -> gate and up products -> SiLU * up -> down product

    python examples/paged_decoder_layer.py
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
    group: int = 64       # of k that share a scale
    page: int = 16
    theta: float = 10000.0
    eps: float = 1e-5


class Weights4:
    """[n, k] weights in 4 bits: bytes [n, k/2], scales and zero points [n, k/group]."""

    def __init__(self, w: torch.Tensor, group: int):
        n, k = w.shape
        g = w.float().view(n, k // group, group)
        lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        self.scales = ((hi - lo).clamp_min(1e-8) / 15).bfloat16()
        s = self.scales.float()
        self.zeros = torch.round(-lo / s).clamp(0, 15).to(torch.uint8)
        q = (torch.round(g / s) + self.zeros.float()).clamp(0, 15).to(torch.uint8).view(n, k)
        self.bytes = (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous()
        self.n, self.k, self.group = n, k, group

    def dense(self) -> torch.Tensor:
        q = torch.stack((self.bytes & 15, self.bytes >> 4), -1).view(self.n, self.k // self.group, self.group).double()
        return ((q - self.zeros.double()) * self.scales.double()).view(self.n, self.k)


class Layer:
    def __init__(self, dev: "hal.CudaSm100Device", c: Config, pages: int, seed: int = 0):
        self.dev, self.c = dev, c
        g = torch.Generator(device="cuda:0")
        g.manual_seed(seed)

        def weights(n, k):
            return Weights4(torch.randn((n, k), generator=g, device="cuda:0") * k ** -0.5, c.group)

        d = c.head_dim
        self.wq, self.wk, self.wv = weights(c.heads_q * d, c.hidden), weights(c.heads_kv * d, c.hidden), weights(c.heads_kv * d, c.hidden)
        self.wo, self.gate, self.up, self.down = weights(c.hidden, c.heads_q * d), weights(c.inner, c.hidden), weights(c.inner, c.hidden), weights(c.hidden, c.inner)
        self.norm1, self.norm2 = ((1 + 0.1 * torch.randn(c.hidden, generator=g, device="cuda:0")).bfloat16() for _ in range(2))
        shape = (pages, c.heads_kv, c.page, d)
        self.k, self.v = (torch.zeros(shape, dtype=torch.int8, device="cuda:0") for _ in range(2))
        self.k_scales, self.v_scales = (torch.zeros(shape[:3], device="cuda:0") for _ in range(2))
        self.cache = hal.PagedKv(capi.I8, c.heads_kv, d, c.page, pages, *(t.data_ptr() for t in (self.k, self.v, self.k_scales, self.v_scales)))

    def _norm(self, x, residual, weight, stream):
        """(x + residual, its norm as whole numbers, their steps)"""
        rows = x.shape[0]
        total, q, steps = torch.empty_like(x), torch.empty_like(x, dtype=torch.int8), torch.empty(rows, device=x.device)
        self.dev.add_rms_norm(capi.BF16, rows, self.c.hidden, self.c.eps, x.data_ptr(), 0 if residual is None else residual.data_ptr(), total.data_ptr(),
                              weight.data_ptr(), q.data_ptr(), out_dtype=capi.I8, scales=steps.data_ptr(), stream=stream)
        return total, q, steps

    def _product(self, a, steps, w, stream):
        out = torch.empty((a.shape[0], w.n), dtype=torch.bfloat16, device=a.device)
        eight = steps is not None
        self.dev.gemm_w4(capi.BF16, a.shape[0], w.n, w.k, w.group, a.data_ptr(), w.bytes.data_ptr(), w.scales.data_ptr(), out.data_ptr(),
                         a_dtype=capi.I8 if eight else capi.BF16, a_scales=steps.data_ptr() if eight else 0, w_zeros=w.zeros.data_ptr(), stream=stream)
        return out

    def step(self, x: torch.Tensor, news: list, lens: list, table: torch.Tensor, lens_d: torch.Tensor, starts_d: torch.Tensor) -> torch.Tensor:
        """x [tokens, hidden] bf16: the new tokens of all sequences, news[b] of the lens[b] positions that sequence b then has."""
        c, dev, st = self.c, self.dev, torch.cuda.current_stream().cuda_stream
        batch = hal.PagedBatch(len(news), x.shape[0], max(news), max(lens), table.shape[1], table.data_ptr(), lens_d.data_ptr(), starts_d.data_ptr())
        h, a, steps = self._norm(x, None, self.norm1, st)
        q, k, v = (self._product(a, steps, w, st) for w in (self.wq, self.wk, self.wv))
        at = 0
        for new, n in zip(news, lens):  # every sequence is at a position of its own
            for t, heads in ((q, c.heads_q), (k, c.heads_kv)):
                if new:
                    dev.rope(capi.BF16, 1, new, heads, c.head_dim, n - new, c.theta, t[at:].data_ptr(), stream=st)
            at += new
        dev.kv_page_append(self.cache, batch, capi.BF16, k.data_ptr(), v.data_ptr(), stream=st)
        o = torch.empty_like(q)
        dev.attention_paged(self.cache, batch, capi.BF16, c.heads_q, q.data_ptr(), o.data_ptr(), stream=st)
        h, a, steps = self._norm(self._product(o, None, self.wo, st), h, self.norm2, st)
        gate, up = (self._product(a, steps, w, st) for w in (self.gate, self.up))
        act = torch.empty_like(gate)
        dev.silu_mul(capi.BF16, x.shape[0], c.inner, gate.data_ptr(), up.data_ptr(), act.data_ptr(), stream=st)
        return self._product(act, None, self.down, st) + h


class Pages:
    """Pages handed to sequences as they grow."""

    def __init__(self, sequences: int, per_sequence: int, page: int):
        self.page, self.free = page, list(range(sequences * per_sequence))[::-1]
        self.table = torch.zeros((sequences, per_sequence), dtype=torch.int32)
        self.held = [0] * sequences

    def grow(self, b: int, length: int) -> None:
        while self.held[b] * self.page < length:
            self.table[b, self.held[b]] = self.free.pop()
            self.held[b] += 1


def serve(layer: Layer, prompts: list, chunk: int, generated: int):
    """Feeds prompts [tokens, hidden] in chunks, one call a step for all sequences, then generates by feeding back the layer's output.  Yields (sequence's new tokens,
    lengths, input, output) of every step."""
    c = layer.c
    most = max(p.shape[0] for p in prompts) + generated
    pages = Pages(len(prompts), -(-most // c.page), c.page)
    done, last = [0] * len(prompts), [None] * len(prompts)
    while any(n < p.shape[0] + generated for n, p in zip(done, prompts)):
        parts, news = [], []
        for b, p in enumerate(prompts):
            if done[b] < p.shape[0]:
                part = p[done[b]:done[b] + chunk]
            elif done[b] < p.shape[0] + generated:
                part = last[b]
            else:
                part = p[:0]
            parts.append(part)
            news.append(part.shape[0])
            done[b] += part.shape[0]
            pages.grow(b, done[b])
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        x = torch.cat(parts)
        table, lens, begin = (torch.as_tensor(t, dtype=torch.int32).to("cuda:0") for t in (pages.table, done, starts))
        y = layer.step(x, news, list(done), table, lens, begin)
        for b, n in enumerate(news):
            if n:
                last[b] = torch.nn.functional.normalize(y[starts[b + 1] - 1:starts[b + 1]].float(), dim=-1).mul(c.hidden ** 0.5).bfloat16()
        yield news, list(done), x, y


def main() -> None:
    c = Config()
    dev = hal.CudaSm100Device(0)
    layer = Layer(dev, c, pages=4 * 80)
    prompts = [torch.randn((n, c.hidden), device="cuda:0").bfloat16() for n in (700, 90, 333, 1)]
    for _ in serve(layer, prompts, chunk=256, generated=2):
        pass
    torch.cuda.synchronize()
    began, tokens, steps = time.perf_counter(), 0, 0
    for news, lens, _, _ in serve(layer, prompts, chunk=256, generated=32):
        tokens, steps = tokens + sum(news), steps + 1
    torch.cuda.synchronize()
    assert dev.status() == 0
    took = time.perf_counter() - began
    print(f"{steps} steps, {tokens} tokens of {len(prompts)} sequences (up to {max(lens)} positions, 8-bit cache, 4-bit weights): {1e3 * took / steps:.2f} ms a step")


if __name__ == "__main__":
    main()
