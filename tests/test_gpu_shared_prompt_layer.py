"""Rows and products in 8 bits, attention behind a shared prompt and cross attention together: the example's layer against the same layer in 64 bits."""
import importlib.util
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "shared_prompt_layer.py"
    spec = importlib.util.spec_from_file_location("shared_prompt_layer", path)
    mod = importlib.util.module_from_spec(spec)
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


def attend(q, k, v, hidden=None):
    group = q.shape[1] // k.shape[1]
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("qhd,khd->hqk", q, k) / q.shape[2] ** 0.5
    if hidden is not None:
        s = s.masked_fill(hidden, -float("inf"))
    return torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v)


def reference(layer, x, first, cache, states):
    """The layer on one sequence's new tokens in 64 bits; cache: its keys and values so far."""
    c = layer.c

    def norm(h, w):
        return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + c.eps) * w.double()

    def heads(t, w, n):
        return (t @ w.dense().T).view(-1, n, c.head_dim)

    a = norm(x, layer.norms[0])
    q, k, v = rotated(heads(a, layer.wq, c.heads_q), first, c.theta), rotated(heads(a, layer.wk, c.heads_kv), first, c.theta), heads(a, layer.wv, c.heads_kv)
    cache = [torch.cat((cache[0], k)), torch.cat((cache[1], v))]
    hidden = torch.arange(cache[0].shape[0], device=x.device)[None] > first + torch.arange(x.shape[0], device=x.device)[:, None]
    h = x + attend(q, *cache, hidden).flatten(1) @ layer.wo.dense().T
    a = norm(h, layer.norms[1])
    o = attend(heads(a, layer.cross_q, c.heads_q), heads(states, layer.cross_k, c.heads_kv), heads(states, layer.cross_v, c.heads_kv))
    h = h + o.flatten(1) @ layer.cross_o.dense().T
    both = norm(h, layer.norms[2]) @ layer.gate_up.dense().T
    gate, up = both[:, :c.inner], both[:, c.inner:]
    return (gate * torch.sigmoid(gate) * up) @ layer.down.dense().T + h, cache


@pytest.mark.parametrize("prompt_len", [150, 1600, 9])
def test_layer(dev, example, prompt_len):
    """A prompt that ends inside a page, one of whole pages, and one that fills none, so that nothing is shared."""
    c = example.Config()
    layer = example.Layer(dev, c, seed=3)
    g = torch.Generator(device="cuda:0")
    g.manual_seed(4)
    prompt, *rest = (torch.randn((n, c.hidden), generator=g, device="cuda:0").bfloat16() for n in (prompt_len, 70, 0, 1, 133, 2, 1, 40, 3))
    states, first = rest[:4], rest[4:]
    empty = [torch.zeros((0, c.heads_kv, c.head_dim), dtype=torch.float64, device="cuda:0") for _ in range(2)]
    whole = prompt_len // c.page * c.page
    caches, shared, steps = None, None, 0
    for step, x, y in example.serve(layer, prompt, states, first, generated=2):
        at = 0
        if caches is None:
            want, cache = reference(layer, x.double(), 0, empty, x[:0].double())
            shared = [t[:whole] for t in cache]
            wants, caches = [want], [shared] * 4
        else:
            wants = []
            for b, new in enumerate(step.news):
                want, caches[b] = reference(layer, x[at:at + new].double(), step.lens[b] - new, caches[b], states[b].double())
                wants.append(want)
                at += new
        at = 0
        for b, want in enumerate(wants):
            # Rows in 8 bits: half a step of 127 of a row's largest, four times its root mean square (eight for gated ones), is 0.5 to 1 % of that (uniform: / sqrt 3) in
            # each of the six; 16-bit roundings are 0.2 %.  Together at most 2 % of the layer's own part, of which x is the larger
            got = y[at:at + want.shape[0]].double()
            off = (got - want).norm() / want.norm()
            assert off <= 0.02, (steps, b, float(off))
            at += want.shape[0]
        steps += 1
    assert steps == 4 and dev.status() == 0
