"""More operators of a serving step and the work they are measured on: products of 8-bit activations with 8-bit weights, the rows in 8 bits that such
products take (of attention's output, or of a gated layer's), attention of a batch whose sequences share a long prefix, and cross attention to the states
of an encoder, both over the pages of a key-value cache.

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
        # a square projection for one token: reading the weights is all there is
        {"name": "i8_bf16_1x4096x4096", "op": "i8", "dtype": "bf16", "m": 1, "n": 4096, "k": 4096},
        # the gated layer's two projections in one product, for a step of 48 sequences
        {"name": "i8_bf16_48x28672x4096", "op": "i8", "dtype": "bf16", "m": 48, "n": 28672, "k": 4096},
        # a prompt of odd length, an odd number of outputs, so that no row of the result but the first starts where a vector does
        {"name": "i8_f16_777x5003x4112", "op": "i8", "dtype": "f16", "m": 777, "n": 5003, "k": 4112},
        # the chunk of a long prompt through the gated layer's projections: the tensor core decides
        {"name": "i8_bf16_8192x28672x4096", "op": "i8", "dtype": "bf16", "m": 8192, "n": 28672, "k": 4096},
        # attention's output of a step of 48 tokens on its way to the output projection
        {"name": "rows_bf16_48x4096", "op": "rows", "dtype": "bf16", "rows": 48, "cols": 4096, "gated": False},
        # a chunk's gated activations, gate and up side by side in the rows of one product, on their way to the down projection
        {"name": "rows_bf16_gated_8192x14336", "op": "rows", "dtype": "bf16", "rows": 8192, "cols": 14336, "gated": True},
        # one token for each of 8 sequences that share a prompt of 2048: launch latency and few rows
        {"name": "prefix_bf16_b8_p2048", "op": "prefix", "dtype": "bf16", "cache": "bf16", "batch": 8, "hq": 32, "hkv": 8, "d": 128, "page": 16, "prefix": 2048,
         "new": 1, "len": 300, "spread": 2},
        # one token for each of 64 sequences on a shared prompt of 16384, 8-bit cache
        {"name": "prefix_i8_b64_p16384", "op": "prefix", "dtype": "bf16", "cache": "i8", "batch": 64, "hq": 32, "hkv": 8, "d": 128, "page": 16, "prefix": 16384,
         "new": 1, "len": 1500, "spread": 3},
        # many sequences on a long shared document
        {"name": "prefix_bf16_b128_p32768", "op": "prefix", "dtype": "bf16", "cache": "bf16", "batch": 128, "hq": 32, "hkv": 8, "d": 128, "page": 64,
         "prefix": 32768, "new": 1, "len": 900, "spread": 5},
        # a few proposed tokens for each of 24 sequences, heads of 64 in groups of seven
        {"name": "prefix_f16_b24_p6016_new5", "op": "prefix", "dtype": "f16", "cache": "f16", "batch": 24, "hq": 28, "hkv": 4, "d": 64, "page": 32, "prefix": 6016,
         "new": 5, "len": 700, "spread": 7},
        # one token for each of 32 sequences, each on its own encoder's states of up to 1500 positions, a head of keys for every head of queries
        {"name": "cross_bf16_b32_s1500", "op": "cross", "dtype": "bf16", "cache": "bf16", "batch": 32, "hq": 16, "hkv": 16, "d": 64, "page": 64, "new": 1,
         "len": 1500, "spread": 11},
        # prompts of up to 448 tokens against encoders of up to 4000 positions, grouped heads; one encoder has nothing to say
        {"name": "cross_f16_b8_448_on_4000", "op": "cross", "dtype": "f16", "cache": "f16", "batch": 8, "hq": 32, "hkv": 8, "d": 128, "page": 32, "new": 448,
         "len": 4000, "spread": 13},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["i8", "i8", "rows", "prefix", "prefix", "cross"])
    half = rng.choice(["bf16", "bf16", "f16"])
    if op == "i8":
        m, n, k = _log(rng, 1, 8192), _log(rng, 64, 28672), _log(rng, 64, 16384)
        kind = rng.random()
        if kind < 0.6:
            n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
        elif kind < 0.9:
            k = max(64, k // 16 * 16)
        while m * n * k > 8e11:
            m = (m + 1) // 2
        return {"op": "i8", "dtype": rng.choice([half, half, half, "f32"]), "m": m, "n": n, "k": k}
    if op == "rows":
        cols = _log(rng, 64, 28672)
        if rng.random() < 0.7:
            cols = max(64, cols // 8 * 8)
        rows = _log(rng, 1, max(2, min(20000, (1 << 26) // cols)))
        return {"op": "rows", "dtype": rng.choice(["f32", half, half, half]), "rows": rows, "cols": cols, "gated": rng.random() < 0.5}
    page, spread = rng.choice([8, 16, 16, 32, 64, 128, 24]), rng.randrange(1, 1 << 20)
    cache, d = rng.choice([half, half, "i8"]), rng.choice([64, 128, 128])
    group, hkv = rng.choice([1, 2, 4, 4, 7, 8]), rng.choice([2, 4, 8])
    if op == "prefix":
        prefix = max(1, _log(rng, 256, 49152) // page) * page
        new = 1 if rng.random() < 0.6 else _log(rng, 2, 64)
        length = new + _log(rng, 1, 3000)
        most = int(min(128, 1.3e8 / (group * hkv * new * (prefix + length)), 4e6 / (length * hkv)))
        return {"op": "prefix", "dtype": half, "cache": cache, "batch": _log(rng, 1, max(2, most)) if most > 1 else 1, "hq": group * hkv, "hkv": hkv, "d": d,
                "page": page, "prefix": prefix, "new": new, "len": length, "spread": spread}
    new = 1 if rng.random() < 0.5 else _log(rng, 2, 512)
    length = _log(rng, 1, 8000)
    most = int(min(64, 1.3e8 / (group * hkv * new * length), 2e6 / (length * hkv)))
    return {"op": "cross", "dtype": half, "cache": cache, "batch": _log(rng, 1, max(2, most)) if most > 1 else 1, "hq": group * hkv, "hkv": hkv, "d": d,
            "page": page, "new": new, "len": length, "spread": spread}


def sequences(case):
    """(new tokens, positions) of every sequence, positions behind the prefix where there is one; the first has the case's own.  A prompt's own positions hold its new
    tokens; an encoder's states are any number, in one sequence of nine none."""
    rng, got = random.Random(case["spread"]), [(case["new"], case["len"])]
    for b in range(1, case["batch"]):
        new = rng.randint(1, case["new"])
        if case["op"] == "prefix":
            got.append((new, rng.randint(new, case["len"])))
        else:
            got.append((new, 0 if b % 9 == 4 else rng.randint(1, case["len"])))
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


def _pages(s, gen, c):
    """A cache in the middle of its life: pages in any order, filled with what tokens before, or an encoder, have left.  Sequences that share a prefix begin with the
    same pages."""
    seqs, ps, d = sequences(c), c["page"], c["d"]
    shared = c.get("prefix", 0) // ps
    need = [-(-n // ps) for _, n in seqs]
    pages = shared + sum(need) + 3
    order, at = torch.randperm(pages, generator=gen, device=GPU).int(), shared
    table = torch.zeros((len(seqs), max(1, shared + max(need))), dtype=torch.int32, device=GPU)
    table[:, :shared] = order[:shared]
    for b, n in enumerate(need):
        table[b, shared:shared + n] = order[at:at + n]
        at += n
    starts = [0]
    for new, _ in seqs:
        starts.append(starts[-1] + new)
    s["table"], s["pages"], s["tokens"] = table, pages, starts[-1]
    s["lens"] = torch.tensor([c.get("prefix", 0) + n for _, n in seqs], dtype=torch.int32, device=GPU)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=GPU)
    for name in ("k", "v"):
        x = _normal(gen, (pages, c["hkv"], ps, d)) * torch.exp(_normal(gen, (pages, c["hkv"], ps, 1), 0.3))
        if c["cache"] == "i8":
            s[name + "_cache"], s[name + "_scales"] = _quantised(x)
        else:
            s[name + "_cache"], s[name + "_scales"] = x.to(TORCH[c["cache"]]), None
        del x


def prepare(case, seed):
    gen = torch.Generator(device=GPU)
    gen.manual_seed(int(seed))
    c = dict(case)
    s, t = {"case": c}, TORCH[c["dtype"]]
    if c["op"] == "i8":
        m, n, k = c["m"], c["n"], c["k"]
        s["a"], s["a_scales"] = _quantised(_activations(gen, (m, k)))
        s["w"], s["w_scales"] = _quantised(_normal(gen, (n, k), k ** -0.5) * torch.exp(_normal(gen, (n, 1), 0.3)))
        s["c"] = torch.empty((m, n), dtype=t, device=GPU)
    elif c["op"] == "rows":
        rows, cols = c["rows"], c["cols"]
        s["x"] = _activations(gen, (rows, 2 * cols if c["gated"] else cols)).to(t)
        s["y"], s["scales"] = torch.empty((rows, cols), dtype=torch.int8, device=GPU), torch.empty(rows, device=GPU)
        s["values"] = torch.empty((rows, cols), dtype=t, device=GPU)
    else:
        _pages(s, gen, c)
        s["q"] = _normal(gen, (s["tokens"], c["hq"], c["d"]), 2.0).to(t)
        s["o"] = torch.empty_like(s["q"])
    if own:  # the device's handle, and for a cache the descriptions that a program keeps beside it
        s["dev"] = device()
        if "table" in s:
            hal = importlib.import_module("tile-rs_b200").hal
            s["kv"] = hal.PagedKv(code(c["cache"]), c["hkv"], c["d"], c["page"], s["pages"], s["k_cache"].data_ptr(), s["v_cache"].data_ptr(),
                                  *(0 if s[x] is None else s[x].data_ptr() for x in ("k_scales", "v_scales")))
            s["step"] = hal.PagedBatch(c["batch"], s["tokens"], c["new"], 0, s["table"].shape[1], s["table"].data_ptr(), s["lens"].data_ptr(),
                                       s["starts"].data_ptr())
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    c, dev, st, t = s["case"], s["dev"], stream(), code(s["case"]["dtype"])
    if c["op"] == "i8":
        dev.gemm_i8(t, c["m"], c["n"], c["k"], s["a"].data_ptr(), s["a_scales"].data_ptr(), s["w"].data_ptr(), s["w_scales"].data_ptr(), s["c"].data_ptr(),
                    stream=st)
        return s["c"]
    if c["op"] == "rows":
        x, cols = s["x"], c["cols"]
        dev.quantise_rows(t, c["rows"], cols, x.data_ptr(), s["y"].data_ptr(), s["scales"].data_ptr(), pitch=x.shape[1],
                          up=x.data_ptr() + cols * x.element_size() if c["gated"] else 0, stream=st)
        return {"y": torch.mul(s["y"], s["scales"][:, None], out=s["values"]), "scales": s["scales"]}
    if c["op"] == "prefix":
        dev.attention_paged_prefix(s["kv"], s["step"], t, c["hq"], c["prefix"], s["table"].data_ptr(), s["q"].data_ptr(), s["o"].data_ptr(), stream=st)
    else:
        dev.attention_paged_cross(s["kv"], s["step"], t, c["hq"], s["q"].data_ptr(), s["o"].data_ptr(), stream=st)
    return s["o"]


def _plain(s):
    c, t = s["case"], TORCH[s["case"]["dtype"]]
    if c["op"] == "i8":
        return ((s["a"].float() @ s["w"].float().T) * s["a_scales"][:, None] * s["w_scales"]).to(t)
    if c["op"] == "rows":
        x = s["x"].float()
        if c["gated"]:
            gate, up = x[:, :c["cols"]], x[:, c["cols"]:]
            x = gate / (1.0 + torch.exp(-gate)) * up
        q, step = _quantised(x)
        return {"y": (q * step[:, None]).to(t), "scales": step}
    # attention: every sequence's tokens and its own positions side by side, up to the longest
    b, new, top, hkv, d, base = c["batch"], c["new"], c["len"], c["hkv"], c["d"], c.get("prefix", 0)
    group, ps = c["hq"] // hkv, c["page"]
    token = torch.arange(s["tokens"], device=GPU)
    seq = torch.searchsorted(s["starts"][1:].contiguous(), token.int(), right=True)
    row = token - s["starts"][seq].long()
    q = torch.zeros((b, new, hkv, group, d), device=GPU)
    q[seq, row] = s["q"].float().view(-1, hkv, group, d) * d ** -0.5
    q = q.permute(0, 2, 3, 1, 4).reshape(b, hkv, group * new, d)
    key = base + torch.arange(top, device=GPU)
    lens = s["lens"].long()
    filled = key < lens[:, None]                                                    # [b, top]
    nth = torch.div(key, ps, rounding_mode="floor").clamp_max(s["table"].shape[1] - 1)
    page = s["table"].long()[:, nth]
    k, v = (_values(s, x, page, (key % ps).expand(b, top)).masked_fill_(~filled[..., None, None], 0.0) for x in ("k", "v"))
    p = torch.matmul(q, k.permute(0, 2, 3, 1)).view(b, hkv, group, new, top)
    if base:  # a token sees its prefix, and of its own positions those up to its own
        last = torch.full((b, new), -1, device=GPU)
        last[seq, row] = lens[seq] - s["starts"][seq + 1].long() + token
        hidden = key > last[..., None]                                              # [b, new, top]
    else:
        hidden = ~filled[:, None].expand(b, new, top)
    p.masked_fill_(hidden[:, None, None], -math.inf)
    p = p.view(b, hkv, group * new, top)
    most = p.amax(-1, keepdim=True)
    if base:  # the rows of all sequences against the prefix at once
        place = torch.arange(base, device=GPU)
        shared = s["table"][0].long()[torch.div(place, ps, rounding_mode="floor")]
        pk, pv = (_values(s, x, shared, place % ps).transpose(0, 1) for x in ("k", "v"))     # [hkv, prefix, d]
        first = torch.matmul(q.transpose(0, 1).reshape(hkv, b * group * new, d), pk.transpose(1, 2))
        most = torch.maximum(most, first.amax(-1).view(hkv, b, group * new, 1).transpose(0, 1))
        first.sub_(most.transpose(0, 1).reshape(hkv, -1, 1)).exp_()
    p.sub_(torch.where(most > -math.inf, most, torch.zeros_like(most))).exp_()
    total, o = p.sum(-1, keepdim=True), torch.matmul(p, v.transpose(1, 2))
    if base:
        total = total + first.sum(-1).view(hkv, b, group * new, 1).transpose(0, 1)
        o = o + torch.matmul(first, pv).view(hkv, b, group * new, d).transpose(0, 1)
    o = (o / torch.where(total > 0, total, torch.ones_like(total))).view(b, hkv, group, new, d)
    return o.permute(0, 3, 1, 2, 4)[seq, row].reshape(s["tokens"], c["hq"], d).to(t)


def _values(s, x, page, at):
    """What the cache holds at (page, place), as f32 [..., heads, d]."""
    got = s[x + "_cache"][page, :, at].float()
    return got if s[x + "_scales"] is None else got * s[x + "_scales"][page, :, at][..., None]


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["op"] == "i8":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k + 4 * m + n * k + 4 * n + m * n * e, "flops": 2 * m * n * k}
    if c["op"] == "rows":
        return {"bytes": c["rows"] * (c["cols"] * (e * (2 if c["gated"] else 1) + 1) + 4), "flops": 0}
    seqs, d = sequences(c), c["d"]
    held = d * SIZE[c["cache"]] + (4 if c["cache"] == "i8" else 0)  # a head's row in the cache
    new, total = sum(n for n, _ in seqs), sum(n for _, n in seqs)
    if c["op"] == "prefix":
        pairs = sum(n * (c["prefix"] + t - n) + n * (n + 1) // 2 for n, t in seqs)
        total += c["prefix"]
    else:
        pairs = sum(n * t for n, t in seqs)
    return {"bytes": 2 * new * c["hq"] * d * e + 2 * total * c["hkv"] * held, "flops": 4 * c["hq"] * d * pairs}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------
def _held(s, x, pages, head, count):
    """The first `count` rows of a head on these pages, one after the other, in 64 bits."""
    rows = s[x + "_cache"][pages.long(), head].double()
    if s[x + "_scales"] is not None:
        rows = rows * s[x + "_scales"][pages.long(), head].double()[..., None]
    return rows.reshape(-1, rows.shape[-1])[:count]


def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    if c["op"] == "i8":
        out, a = torch.empty((c["m"], c["n"]), dtype=torch.float64, device=GPU), s["a"].double()
        for g in range(0, c["n"], 4096):
            out[:, g:g + 4096] = a @ s["w"][g:g + 4096].double().T
        out *= s["a_scales"].double()[:, None]
        out *= s["w_scales"].double()[None]
        return out
    if c["op"] == "rows":
        y, scales = torch.empty((c["rows"], c["cols"]), dtype=torch.float64, device=GPU), torch.empty(c["rows"], dtype=torch.float64, device=GPU)
        for r in range(0, c["rows"], 1024):
            x = s["x"][r:r + 1024].double()
            if c["gated"]:
                x = x[:, :c["cols"]] * torch.sigmoid(x[:, :c["cols"]]) * x[:, c["cols"]:]
            step = x.abs().amax(-1) / 127.0
            scales[r:r + 1024] = step
            y[r:r + 1024] = torch.round(x / step.clamp_min(1e-300)[:, None]) * step[:, None]
        return {"y": y, "scales": scales}
    out, first, group = torch.zeros(s["q"].shape, dtype=torch.float64, device=GPU), 0, c["hq"] // c["hkv"]
    base, ps = c.get("prefix", 0), c["page"]
    common = [[_held(s, x, s["table"][0, :base // ps], g, base) for g in range(c["hkv"])] for x in ("k", "v")]
    for b, (new, n) in enumerate(sequences(c)):
        mine = s["table"][b, base // ps:base // ps + -(-n // ps)]
        own_place = torch.arange(n, device=GPU)[None]
        for g in range(c["hkv"]):
            if base + n == 0:
                continue  # nothing to see: zeros
            k, v = (torch.cat((common[i][g], _held(s, x, mine, g, n))) for i, x in enumerate(("k", "v")))
            q = s["q"][first:first + new, g * group:(g + 1) * group].double()
            score = torch.einsum("thd,kd->htk", q, k) / math.sqrt(c["d"])
            if base:
                score[..., base:].masked_fill_(own_place > torch.arange(n - new, n, device=GPU)[:, None], -math.inf)
            out[first:first + new, g * group:(g + 1) * group] = torch.einsum("htk,kd->thd", torch.softmax(score, -1), v)
        first += new
    return out
