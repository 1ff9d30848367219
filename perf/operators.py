"""The serving operators of this library and the work they are measured on: a norm that adds the residual and may answer in 8 bits, products
with 4-bit weights, a paged key-value cache that may be held in 8 bits, and attention of new tokens over its pages.

Each case is one pass through one of them.  ``own`` picks between the library's kernels and the plain form in elementary torch operations.
``listed()`` names the cases, ``draw()`` picks others of the same ranges, ``exact()`` evaluates the definitions in 64 bits.
"""
import importlib
import math
import random

import torch

own = False  # True: run() calls the library's operators

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}
GPU = "cuda:0"
EPS = 1e-5
#: an 8-bit value is a whole number of 1/127ths of the largest magnitude of its row
STEP = 1.0 / 127.0

_DEVICE = None


def device():
    """One open device per process, as a program of this library keeps it."""
    global _DEVICE
    if _DEVICE is None:
        _DEVICE = importlib.import_module("tile-rs_b200").hal.CudaSm100Device(0)
    return _DEVICE


def code(name):
    capi = importlib.import_module("tile-rs_b200").capi
    return {"f32": capi.F32, "bf16": capi.BF16, "f16": capi.F16, "i8": capi.I8}[name]


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- the cases --------------------------------------------------------------------------------------------------
def listed():
    return [
        # the norm before a projection, one token of one sequence: all of it is launch latency
        {"name": "norm_bf16_1x4096", "op": "norm", "dtype": "bf16", "out": "bf16", "rows": 1, "cols": 4096, "residual": True, "weight": True},
        # the same for a prompt, with the 8-bit rows that the product behind it takes
        {"name": "norm_bf16_i8_8192x4096", "op": "norm", "dtype": "bf16", "out": "i8", "rows": 8192, "cols": 4096, "residual": True, "weight": True},
        # f32 rows of odd length, none of which starts where a vector does
        {"name": "norm_f32_3000x5001", "op": "norm", "dtype": "f32", "out": "f32", "rows": 3000, "cols": 5001, "residual": True, "weight": False},
        # a square projection for one token: reading the weights is all there is
        {"name": "w4_bf16_1x4096x4096", "op": "w4", "dtype": "bf16", "a": "bf16", "m": 1, "n": 4096, "k": 4096, "group": 128, "zeros": False},
        # the gated layer's projection for a step of 16 sequences, on the norm's 8-bit rows
        {"name": "w4_bf16_i8_16x16384x4096", "op": "w4", "dtype": "bf16", "a": "i8", "m": 16, "n": 16384, "k": 4096, "group": 128, "zeros": False},
        # a short prompt through weights with zero points in small groups, an odd number of outputs
        {"name": "w4_f16_200x5003x2048", "op": "w4", "dtype": "f16", "a": "f16", "m": 200, "n": 5003, "k": 2048, "group": 32, "zeros": True},
        # one new token for each of 48 sequences into an 8-bit cache, which is then read back
        {"name": "cache_i8_48x1", "op": "cache", "dtype": "bf16", "cache": "i8", "batch": 48, "heads": 8, "d": 128, "page": 16, "new": 1, "len": 300,
         "spread": 3},
        # chunks of four prompts into an 8-bit cache of large pages, read back with all that came before
        {"name": "cache_i8_4x2048", "op": "cache", "dtype": "bf16", "cache": "i8", "batch": 4, "heads": 8, "d": 128, "page": 64, "new": 2048, "len": 16000,
         "spread": 5},
        # one generated token of one long sequence
        {"name": "paged_bf16_b1_s32768", "op": "paged", "dtype": "bf16", "cache": "bf16", "batch": 1, "hq": 32, "hkv": 8, "d": 128, "page": 64, "new": 1,
         "len": 32768, "spread": 0},
        # one generated token for each of 64 sequences of uneven length, 8-bit cache
        {"name": "paged_i8_b64_s6000", "op": "paged", "dtype": "bf16", "cache": "i8", "batch": 64, "hq": 32, "hkv": 8, "d": 128, "page": 16, "new": 1,
         "len": 6000, "spread": 7},
        # one chunk of a long prompt: everything before it and its own part below the diagonal
        {"name": "paged_bf16_512_on_15872", "op": "paged", "dtype": "bf16", "cache": "bf16", "batch": 1, "hq": 32, "hkv": 8, "d": 128, "page": 64, "new": 512,
         "len": 16384, "spread": 0},
        # a mixed step: chunks and single tokens side by side, heads of 64 in groups of seven, 8-bit cache
        {"name": "paged_f16_i8_mixed", "op": "paged", "dtype": "f16", "cache": "i8", "batch": 12, "hq": 28, "hkv": 4, "d": 64, "page": 32, "new": 600,
         "len": 4000, "spread": 11},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = _any(rng)
    return draw(rng) if 3072 in case.values() else case


def _any(rng):
    op = rng.choice(["norm", "w4", "w4", "cache", "paged", "paged"])
    half = rng.choice(["bf16", "bf16", "f16"])
    if op == "norm":
        dtype, cols = rng.choice(["f32", half, half]), _log(rng, 64, 16384)
        if rng.random() < 0.7:
            cols = max(64, cols // 8 * 8)
        rows = _log(rng, 1, max(2, min(20000, (1 << 25) // cols)))
        return {"op": "norm", "dtype": dtype, "out": rng.choice([dtype, "i8"]), "rows": rows, "cols": cols, "residual": rng.random() < 0.8,
                "weight": rng.random() < 0.8}
    if op == "w4":
        group = rng.choice([32, 64, 128, 128])
        m, n, k = _log(rng, 1, 400), _log(rng, 64, 16384), group * _log(rng, 2, 8192 // group)
        if rng.random() < 0.7:
            n = max(64, n // 16 * 16)
        return {"op": "w4", "dtype": half, "a": rng.choice([half, "i8"]), "m": m, "n": n, "k": k, "group": group, "zeros": rng.random() < 0.3}
    page, spread = rng.choice([8, 16, 16, 32, 64, 128, 24]), rng.randrange(1, 1 << 20)
    cache = rng.choice([half, "i8"])
    d = rng.choice([64, 128, 128])
    if op == "cache":
        new = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
        length = new + _log(rng, 1, 16000)
        heads = rng.choice([1, 2, 4, 8])
        return {"op": "cache", "dtype": half, "cache": cache, "batch": _log(rng, 1, max(2, min(128, 400000 // (length * heads)))), "heads": heads, "d": d,
                "page": page, "new": new, "len": length, "spread": spread}
    group, hkv = rng.choice([1, 2, 4, 4, 5, 8]), rng.choice([2, 4, 8])
    if rng.random() < 0.5:  # single tokens
        length = _log(rng, 1, 40000)
        batch = _log(rng, 1, max(2, min(128, 3000000 // (length * hkv))))
        return {"op": "paged", "dtype": half, "cache": cache, "batch": batch, "hq": group * hkv, "hkv": hkv, "d": d, "page": page, "new": 1, "len": length,
                "spread": spread}
    new = _log(rng, 2, 1024)
    length = new + _log(rng, 1, 12000)
    most = min(16, int(2.5e8 / (group * hkv * new * length)))
    return {"op": "paged", "dtype": half, "cache": cache, "batch": _log(rng, 1, max(2, most)) if most > 1 else 1, "hq": group * hkv, "hkv": hkv, "d": d,
            "page": page, "new": new, "len": length, "spread": spread}


def sequences(case):
    """(new tokens, positions with them) of every sequence: the case's own ones if "spread" is 0 or there is one sequence, else the first has them
    and the others anything down to one new token and no position before it."""
    if case["batch"] == 1 or case["spread"] == 0:
        return [(case["new"], case["len"])] * case["batch"]
    rng, got = random.Random(case["spread"]), [(case["new"], case["len"])]
    for _ in range(case["batch"] - 1):
        new = 1 if rng.random() < 0.4 else rng.randint(1, case["new"])
        got.append((new, rng.randint(new, max(new, case["len"]))))
    return got


# ---- inputs -----------------------------------------------------------------------------------------------------
def _normal(gen, shape, sigma=1.0):
    return torch.randn(shape, generator=gen, device=GPU) * sigma


def _quantised(x):
    """Rows of x as whole numbers of steps of their largest magnitude, and the steps."""
    step = x.abs().amax(-1, keepdim=True) * STEP
    return torch.round(torch.where(step > 0, x / step, torch.zeros_like(x))).to(torch.int8), step.squeeze(-1)


def _activations(gen, shape):
    """Rows with a few columns that stand out, as those of a trained model do."""
    x = _normal(gen, shape)
    x[..., ::97] *= 6.0
    return x


def _pages(s, gen, case, heads):
    """A cache in the middle of its life: pages in any order, filled with what tokens before have left."""
    seqs, ps, d = sequences(case), case["page"], case["d"]
    need = [-(-n // ps) for _, n in seqs]
    pages = sum(need) + 3
    order, table, at = torch.randperm(pages, generator=gen, device=GPU).int(), torch.zeros((len(seqs), max(need)), dtype=torch.int32, device=GPU), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for new, _ in seqs:
        starts.append(starts[-1] + new)
    s["table"], s["pages"], s["tokens"] = table, pages, starts[-1]
    s["lens"] = torch.tensor([n for _, n in seqs], dtype=torch.int32, device=GPU)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=GPU)
    for name in ("k", "v"):
        x = _normal(gen, (pages, heads, ps, d)) * torch.exp(_normal(gen, (pages, heads, ps, 1), 0.3))
        if case["cache"] == "i8":
            s[name + "_cache"], s[name + "_scales"] = _quantised(x)
        else:
            s[name + "_cache"], s[name + "_scales"] = x.to(TORCH[case["cache"]]), None
        del x


def prepare(case, seed):
    gen = torch.Generator(device=GPU)
    gen.manual_seed(int(seed))
    c = dict(case)
    s, t = {"case": c}, TORCH[c["dtype"]]
    if c["op"] == "norm":
        shape = (c["rows"], c["cols"])
        s["x"], s["y"] = _activations(gen, shape).to(t), torch.empty(shape, dtype=torch.int8 if c["out"] == "i8" else t, device=GPU)
        s["residual"] = (4 * _activations(gen, shape)).to(t) if c["residual"] else None
        s["sum"] = torch.empty_like(s["x"]) if c["residual"] else None
        s["weight"] = (1 + _normal(gen, (c["cols"],), 0.2)).to(t) if c["weight"] else None
        s["scales"] = torch.empty(c["rows"], device=GPU) if c["out"] == "i8" else None
        s["values"] = torch.empty(shape, dtype=t, device=GPU) if c["out"] == "i8" else None
    elif c["op"] == "w4":
        m, n, k, groups = c["m"], c["n"], c["k"], c["k"] // c["group"]
        x = _activations(gen, (m, k))
        s["a"], s["a_scales"] = _quantised(x) if c["a"] == "i8" else (x.to(t), None)
        s["w"] = torch.randint(0, 256, (n, k // 2), generator=gen, device=GPU, dtype=torch.uint8)
        s["w_scales"] = (torch.exp(_normal(gen, (n, groups), 0.3)) * (0.25 * k ** -0.5)).to(t)
        s["w_zeros"] = torch.randint(6, 11, (n, groups), generator=gen, device=GPU, dtype=torch.uint8) if c["zeros"] else None
        s["c"] = torch.empty((m, n), dtype=t, device=GPU)
    elif c["op"] == "cache":
        _pages(s, gen, c, c["heads"])
        s["k"], s["v"] = ((_normal(gen, (s["tokens"], c["heads"], c["d"]))).to(t) for _ in range(2))
        # what is read back: every position of every sequence
        places = [0]
        for _, n in sequences(c):
            places.append(places[-1] + n)
        s["places"], s["positions"] = torch.tensor(places, dtype=torch.int32, device=GPU), places[-1]
        s["k_read"], s["v_read"] = (torch.empty((places[-1], c["heads"], c["d"]), dtype=t, device=GPU) for _ in range(2))
    else:
        _pages(s, gen, c, c["hkv"])
        s["q"] = _normal(gen, (s["tokens"], c["hq"], c["d"]), 2.0).to(t)
        s["o"] = torch.empty_like(s["q"])
    if own:  # the device's handle, and for a cache the descriptions that a program keeps beside it
        s["dev"] = device()
        if "table" in s:
            hal, heads = importlib.import_module("tile-rs_b200").hal, c["heads"] if c["op"] == "cache" else c["hkv"]
            s["kv"] = hal.PagedKv(code(c["cache"]), heads, c["d"], c["page"], s["pages"], s["k_cache"].data_ptr(), s["v_cache"].data_ptr(),
                                  *(0 if s[x] is None else s[x].data_ptr() for x in ("k_scales", "v_scales")))
            s["step"] = hal.PagedBatch(c["batch"], s["tokens"], c["new"], c["len"], s["table"].shape[1], s["table"].data_ptr(), s["lens"].data_ptr(),
                                       s["starts"].data_ptr())
            if c["op"] == "cache":
                s["all"] = hal.PagedBatch(c["batch"], s["positions"], c["len"], c["len"], s["table"].shape[1], s["table"].data_ptr(), s["lens"].data_ptr(),
                                          s["places"].data_ptr())
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------
def _at(x):
    return 0 if x is None else x.data_ptr()


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    c, dev, st, t = s["case"], s["dev"], stream(), code(s["case"]["dtype"])
    if c["op"] == "norm":
        dev.add_rms_norm(t, c["rows"], c["cols"], EPS, s["x"].data_ptr(), _at(s["residual"]), _at(s["sum"]), _at(s["weight"]), s["y"].data_ptr(),
                         out_dtype=code(c["out"]), scales=_at(s["scales"]), stream=st)
        if c["out"] == "i8":
            return {"y": torch.mul(s["y"], s["scales"][:, None], out=s["values"]), "scales": s["scales"], "sum": s["sum"]}
        return {"y": s["y"], "sum": s["sum"]}
    if c["op"] == "w4":
        dev.gemm_w4(t, c["m"], c["n"], c["k"], c["group"], s["a"].data_ptr(), s["w"].data_ptr(), s["w_scales"].data_ptr(), s["c"].data_ptr(),
                    a_dtype=code(c["a"]), a_scales=_at(s["a_scales"]), w_zeros=_at(s["w_zeros"]), stream=st)
        return s["c"]
    if c["op"] == "cache":
        dev.kv_page_append(s["kv"], s["step"], t, s["k"].data_ptr(), s["v"].data_ptr(), stream=st)
        dev.kv_page_read(s["kv"], s["all"], t, s["k_read"].data_ptr(), s["v_read"].data_ptr(), stream=st)
        return {"k": s["k_read"], "v": s["v_read"]}
    dev.attention_paged(s["kv"], s["step"], t, c["hq"], s["q"].data_ptr(), s["o"].data_ptr(), stream=st)
    return s["o"]


def _rows(starts, lens, count):
    """For `count` tokens, dealt to sequences by `starts`: the sequence of each and its position in it."""
    token = torch.arange(count, device=GPU)
    seq = torch.searchsorted(starts[1:].contiguous(), token.int(), right=True)
    return seq, lens[seq].long() - starts[seq + 1].long() + token


def _place(s, seq, pos):
    ps = s["case"]["page"]
    return s["table"][seq, torch.div(pos, ps, rounding_mode="floor")].long(), pos % ps


def _plain(s):
    c, t = s["case"], TORCH[s["case"]["dtype"]]
    if c["op"] == "norm":
        h = s["x"].float()
        if c["residual"]:
            h = h + s["residual"].float()
            s["sum"].copy_(h)
        r = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
        z = h * s["weight"].float() if c["weight"] else h
        if c["out"] != "i8":
            return {"y": (z * r).to(t), "sum": s["sum"]}
        # the step of the row before it is normalised: the whole numbers do not depend on how the squares were summed
        step = z.abs().amax(-1, keepdim=True) * STEP
        q = torch.round(torch.where(step > 0, z / step, torch.zeros_like(z)))
        scales = step * r
        return {"y": (q * scales).to(t), "scales": scales.squeeze(-1), "sum": s["sum"]}
    if c["op"] == "w4":
        n, k, g = c["n"], c["k"], c["group"]
        w = torch.stack((s["w"] & 15, s["w"] >> 4), -1).view(n, k // g, g).float()
        w = (w - (s["w_zeros"][..., None].float() if c["zeros"] else 8.0)) * s["w_scales"][..., None].float()
        a = s["a"].float()
        if c["a"] == "i8":
            a = a * s["a_scales"][:, None]
        return (a @ w.view(n, k).T).to(t)
    if c["op"] == "cache":
        page, at = _place(s, *_rows(s["starts"], s["lens"], s["tokens"]))
        pages, places = _place(s, *_rows(s["places"], s["lens"], s["positions"]))
        return {x: _through(s, x, page, at, pages, places).to(t) for x in ("k", "v")}
    # attention: every sequence's tokens and positions side by side, up to the longest
    b, new, top, hkv, d = c["batch"], c["new"], c["len"], c["hkv"], c["d"]
    group = c["hq"] // hkv
    seq, pos = _rows(s["starts"], s["lens"], s["tokens"])
    row = torch.arange(s["tokens"], device=GPU) - s["starts"][seq].long()
    q = torch.zeros((b, new, hkv, group, d), device=GPU)
    q[seq, row] = s["q"].float().view(-1, hkv, group, d)
    key = torch.arange(top, device=GPU)
    filled = key < s["lens"][:, None]                                               # [b, top]
    page = s["table"].long().gather(1, torch.div(key, c["page"], rounding_mode="floor").expand(b, top).contiguous())
    k, v = (_values(s, x, page, (key % c["page"]).expand(b, top)).masked_fill_(~filled[..., None, None], 0.0) for x in ("k", "v"))
    p = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(b, hkv, group * new, d), k.permute(0, 2, 3, 1)).mul_(d ** -0.5).view(b, hkv, group, new, top)
    sees = torch.full((b, new), -1, device=GPU)
    sees[seq, row] = pos
    hidden = key > sees[..., None]                                                  # [b, new, top]
    p.masked_fill_(hidden[:, None, None], -math.inf)
    most = p.amax(-1, keepdim=True)
    p.sub_(torch.where(most > -math.inf, most, torch.zeros_like(most))).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hkv, group * new, top), v.transpose(1, 2)).view(b, hkv, group, new, d) / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4)[seq, row].reshape(s["tokens"], c["hq"], d).to(t)


def _values(s, x, page, at):
    """What the cache holds at (page, place), as f32 [..., heads, d]."""
    got = s[x + "_cache"][page, :, at].float()
    return got if s[x + "_scales"] is None else got * s[x + "_scales"][page, :, at][..., None]


def _through(s, x, page, at, pages, places):
    """The tokens written to the cache, and the cache read back."""
    if s["case"]["cache"] == "i8":
        s[x + "_cache"][page, :, at], s[x + "_scales"][page, :, at] = _quantised(s[x].float())
    else:
        s[x + "_cache"][page, :, at] = s[x]
    return _values(s, x, pages, places)


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["op"] == "norm":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (e * (3 if c["residual"] else 1) + SIZE[c["out"]]) + (e * c["cols"] if c["weight"] else 0) + (4 * c["rows"] if c["out"] == "i8" else 0),
                "flops": 0}
    if c["op"] == "w4":
        m, n, k, groups = c["m"], c["n"], c["k"], c["k"] // c["group"]
        return {"bytes": m * k * SIZE[c["a"]] + (4 * m if c["a"] == "i8" else 0) + n * k // 2 + n * groups * (e + (1 if c["zeros"] else 0)) + m * n * e,
                "flops": 2 * m * n * k}
    seqs, d = sequences(c), c["d"]
    held = d * SIZE[c["cache"]] + (4 if c["cache"] == "i8" else 0)  # a head's row in the cache
    new, total = sum(n for n, _ in seqs), sum(n for _, n in seqs)
    if c["op"] == "cache":
        return {"bytes": 2 * c["heads"] * (new * (d * e + held) + total * (held + d * e)), "flops": 0}
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in seqs)
    return {"bytes": 2 * new * c["hq"] * d * e + 2 * total * c["hkv"] * held, "flops": 4 * c["hq"] * d * pairs}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------
def _held(s, x, b, head, count):
    """The first `count` rows of a head of sequence b, page by page, in 64 bits."""
    ps, got = s["case"]["page"], []
    for i in range(-(-count // ps)):
        page = int(s["table"][b, i])
        rows = s[x + "_cache"][page, head].double()
        got.append(rows if s[x + "_scales"] is None else rows * s[x + "_scales"][page, head].double()[:, None])
    return torch.cat(got)[:count]


def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    if c["op"] == "norm":
        h = s["x"].double() + (s["residual"].double() if c["residual"] else 0.0)
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / c["cols"] + EPS)
        if c["weight"]:
            y = y * s["weight"].double()
        total = h if c["residual"] else None
        if c["out"] != "i8":
            return {"y": y, "sum": total}
        scales = y.abs().amax(-1) / 127.0
        steps = torch.round(y / scales.clamp_min(1e-300)[:, None])
        return {"y": steps * scales[:, None], "scales": scales, "sum": total}
    if c["op"] == "w4":
        out, a = torch.empty((c["m"], c["n"]), dtype=torch.float64, device=GPU), s["a"].double()
        if c["a"] == "i8":
            a *= s["a_scales"].double()[:, None]
        for g in range(0, c["n"], 4096):
            w = torch.empty((min(4096, c["n"] - g), c["k"]), dtype=torch.float64, device=GPU)
            w[:, 0::2], w[:, 1::2] = (s["w"][g:g + 4096] % 16).double(), torch.div(s["w"][g:g + 4096], 16, rounding_mode="floor").double()
            zero = s["w_zeros"][g:g + 4096].double() if c["zeros"] else torch.full((w.shape[0], c["k"] // c["group"]), 8.0, dtype=torch.float64, device=GPU)
            w = (w - zero.repeat_interleave(c["group"], 1)) * s["w_scales"][g:g + 4096].double().repeat_interleave(c["group"], 1)
            out[:, g:g + 4096] = a @ w.T
        return out
    seqs = sequences(c)
    if c["op"] == "cache":
        got, at = {}, [0]
        for _, n in seqs:
            at.append(at[-1] + n)
        for x in ("k", "v"):
            out, first = torch.empty((at[-1], c["heads"], c["d"]), dtype=torch.float64, device=GPU), 0
            for b, (new, n) in enumerate(seqs):
                for h in range(c["heads"]):
                    out[at[b]:at[b + 1], h] = _held(s, x, b, h, n)
                fresh = s[x][first:first + new].double()
                if c["cache"] == "i8":
                    step = fresh.abs().amax(-1, keepdim=True) / 127.0
                    fresh = torch.round(fresh / step.clamp_min(1e-300)) * step
                out[at[b + 1] - new:at[b + 1]] = fresh
                first += new
            got[x] = out
        return got
    out, first, group = torch.empty(s["q"].shape, dtype=torch.float64, device=GPU), 0, c["hq"] // c["hkv"]
    for b, (new, n) in enumerate(seqs):
        last = torch.arange(n - new, n, device=GPU)[:, None]
        place = torch.arange(n, device=GPU)[None]
        for g in range(c["hkv"]):
            k, v = _held(s, "k", b, g, n), _held(s, "v", b, g, n)
            for h in range(g * group, (g + 1) * group):
                score = s["q"][first:first + new, h].double() @ k.T / math.sqrt(c["d"])
                out[first:first + new, h] = torch.softmax(score.masked_fill(place > last, -math.inf), -1) @ v
        first += new
    return out
