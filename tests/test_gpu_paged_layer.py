"""The serving operators together: the example's decoder layer, prompts in chunks and single tokens side by side, against the same layer in 64 bits."""
import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "paged_decoder_layer.py"
    spec = importlib.util.spec_from_file_location("paged_decoder_layer", path)
    mod = importlib.util.module_from_spec(spec)
    import sys
    sys.modules[spec.name] = mod  # dataclasses look their module up
    spec.loader.exec_module(mod)
    return mod


def rotated(x, first, theta):
    n, _, d = x.shape
    freq = theta ** (-torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / d)
    angle = (first + torch.arange(n, dtype=torch.float64, device=x.device))[:, None] * freq
    co, si = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * co - b * si, a * si + b * co), -1).reshape(x.shape)


def reference(layer, c, x, first, cache):
    """The layer on one sequence's new tokens in 64 bits; cache: its keys and values so far."""
    def norm(h, w):
        return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + c.eps) * w.double()

    a = norm(x, layer.norm1)
    q, k, v = (a @ w.dense().T for w in (layer.wq, layer.wk, layer.wv))
    q, k, v = q.view(-1, c.heads_q, c.head_dim), k.view(-1, c.heads_kv, c.head_dim), v.view(-1, c.heads_kv, c.head_dim)
    q, k = rotated(q, first, c.theta), rotated(k, first, c.theta)
    cache[0], cache[1] = torch.cat((cache[0], k)), torch.cat((cache[1], v))
    kk, vv = (t.repeat_interleave(c.heads_q // c.heads_kv, 1) for t in cache)
    s = torch.einsum("qhd,khd->hqk", q, kk) / c.head_dim ** 0.5
    hidden = torch.arange(kk.shape[0], device=x.device)[None] > first + torch.arange(x.shape[0], device=x.device)[:, None]
    o = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(hidden, -float("inf")), -1), vv).reshape(x.shape[0], -1)
    h = x + o @ layer.wo.dense().T
    a = norm(h, layer.norm2)
    gate, up = a @ layer.gate.dense().T, a @ layer.up.dense().T
    return (torch.nn.functional.silu(gate) * up) @ layer.down.dense().T + h


def test_layer(dev, example):
    c = example.Config()
    layer = example.Layer(dev, c, pages=4 * 16, seed=3)
    g = torch.Generator(device="cuda:0")
    g.manual_seed(4)
    prompts = [torch.randn((n, c.hidden), generator=g, device="cuda:0").bfloat16() for n in (200, 31, 100, 1)]
    caches = [[torch.zeros((0, c.heads_kv, c.head_dim), dtype=torch.float64, device="cuda:0") for _ in range(2)] for _ in prompts]
    steps = 0
    for news, lens, x, y in example.serve(layer, prompts, chunk=64, generated=3):
        at = 0
        for b, (new, n) in enumerate(zip(news, lens)):
            if new:
                want = reference(layer, c, x[at:at + new].double(), n - new, caches[b])
                # 8-bit rows and cache: half a step of 127 of a row's largest, which is about four times its root mean square, is 0.9 % of that (uniform: / sqrt 3) in each of
                # the norms' rows, K and V; 16-bit roundings are 0.2 %.  All together about 1.5 % of the layer's own part, of which x is the larger
                off = (y[at:at + new].double() - want).norm() / want.norm()
                assert off <= 0.02, (steps, b, float(off))
            at += new
        steps += 1
    assert steps == 7 and dev.status() == 0
