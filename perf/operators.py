"""Attention of windowed models over the paged cache: what a layer calls, and its plain form.

Three operators that a windowed model's attention needs beside the ones this framework has:

``append``   the per-head RMS norms of queries and keys, the position rotation (one position or
             several axes) and the write of keys and values into their pages, straight from the
             rows of the stacked Q/K/V product;
``decode``   one new token per sequence over a sliding window and the first tokens (sinks);
``prefill``  a prompt chunk whose every token has a window of its own, and the sinks.

``step`` is a decode step as it is used: the append, then the attention that reads it.

With ``own`` false ``run`` computes them with elementary torch operations in 32 bits (angles in 64);
with ``own`` true it calls the framework.  A Q8_0 pool is measured through ``step`` and ``prefill``,
whose attention reads it: decoding its bytes would be no part of an append.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
PAGE = 256
# query heads, kv heads, head_dim
SHAPES = {"mixtral": (32, 8, 128), "half": (16, 4, 128), "even": (16, 16, 64), "tiny": (8, 4, 32)}
KV_TYPE = {"f32": 0, "f16": 1, "q8_0": 8}
ROW = {"f32": 4.0, "f16": 2.0, "q8_0": 34.0 / 32.0}  # cache bytes an element


def listed():
    return [
        # the newest token of one conversation: launches and latency
        {"name": "norm_token", "op": "append", "kv": "f16", "shape": "mixtral", "past": 4095, "n_tok": 1,
         "norm": True, "axes": "", "mix": False, "neox": True, "rot": 128},
        # a prompt chunk with normed heads
        {"name": "norm_chunk", "op": "append", "kv": "f16", "shape": "mixtral", "past": 2048, "n_tok": 2048,
         "norm": True, "axes": "", "mix": False, "neox": True, "rot": 128},
        # a prompt with a picture in it: time, height and width in blocks of pairs
        {"name": "axes_picture", "op": "append", "kv": "f16", "shape": "half", "past": 77, "n_tok": 1733,
         "norm": False, "axes": "16,24,24", "mix": False, "neox": True, "rot": 128},
        # a long video prompt into the cache type of 32 bits, axes dealt in turn, heads normed
        {"name": "axes_video_f32", "op": "append", "kv": "f32", "shape": "mixtral", "past": 0, "n_tok": 8192,
         "norm": True, "axes": "24,20,20", "mix": True, "neox": True, "rot": 128},
        # a small model's short conversations, one just begun: the smallest attention
        {"name": "decode_f32_tiny", "op": "decode", "kv": "f32", "shape": "tiny", "lens": "1,700,33,260",
         "window": 256, "sink": 4},
        # one long conversation
        {"name": "decode_f16_b1", "op": "decode", "kv": "f16", "shape": "mixtral", "lens": "30011",
         "window": 4096, "sink": 4},
        # a full serving batch
        {"name": "decode_f16_b64", "op": "decode", "kv": "f16", "shape": "mixtral",
         "lens": ",".join(str(5000 + 1237 * i) for i in range(64)), "window": 4096, "sink": 4},
        # a step of a ragged batch over a quantised cache, the append in it
        {"name": "step_q8_0_b8", "op": "step", "kv": "q8_0", "shape": "mixtral",
         "lens": "8211,30720,12001,5333,17000,32768,9999,21470", "window": 8192, "sink": 16},
        # a chunk of a long prompt: the largest
        {"name": "prefill_f16_4096", "op": "prefill", "kv": "f16", "shape": "mixtral", "past": 8192, "n_tok": 4096,
         "window": 4096, "sink": 4},
        # a chat turn: a short question late in a conversation
        {"name": "prefill_f16_turn", "op": "prefill", "kv": "f16", "shape": "mixtral", "past": 20100, "n_tok": 93,
         "window": 4096, "sink": 4},
        # a ragged chunk over a quantised cache
        {"name": "prefill_q8_0_chunk", "op": "prefill", "kv": "q8_0", "shape": "mixtral", "past": 6000, "n_tok": 777,
         "window": 1024, "sink": 64},
        # a first prompt over the cache type of 32 bits
        {"name": "prefill_f32_first", "op": "prefill", "kv": "f32", "shape": "half", "past": 0, "n_tok": 1500,
         "window": 512, "sink": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "decode", "decode", "step", "prefill", "prefill"])
    shape = rng.choice(["mixtral", "mixtral", "half", "even", "tiny"])
    hd = SHAPES[shape][2]
    if op == "append":
        rot = rng.choice([hd, hd, hd // 2])
        axes = rng.choice(["", "3", "3", "2"])
        if axes == "3":
            a = rng.randint(1, rot // 6)
            b = rng.randint(1, rot // 6)
            axes = "%d,%d,%d" % (rot // 2 - a - b, a, b)
        elif axes == "2":
            a = rng.randint(1, rot // 4)
            axes = "%d,%d" % (rot // 2 - a, a)
        return {"op": op, "kv": rng.choice(["f16", "f16", "f32"]), "shape": shape, "past": rng.randint(0, 30000),
                "n_tok": rng.choice([1, _log(rng, 2, 8000), _log(rng, 2, 8000)]), "norm": rng.random() < 0.6,
                "axes": axes, "mix": rng.random() < 0.5, "neox": rng.random() < 0.7, "rot": rot}
    window = rng.choice([_log(rng, 16, 4096), _log(rng, 16, 8192)])
    sink = rng.choice([0, rng.randint(1, 8), rng.randint(1, 128)])
    kv = rng.choice(["f16", "f16", "f32", "q8_0"])
    if kv == "q8_0" and hd < 64:
        kv = "f16"
    if op == "prefill":
        return {"op": op, "kv": kv, "shape": shape, "past": rng.choice([0, _log(rng, 1, 40000)]),
                "n_tok": _log(rng, 2, 3800), "window": min(window, 4096), "sink": sink}
    lo = 500 if op == "step" else 1  # a step's newest row is one of many, as roundings into 8 bits have it
    lens = [_log(rng, lo, 60000) for _ in range(rng.choice([1, _log(rng, 2, 30)]))]
    return {"op": op, "kv": kv, "shape": shape, "lens": ",".join(map(str, lens)),
            "window": max(window, 500) if op == "step" else window, "sink": sink}


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


def _seen(n, window, sink):
    """Positions that the token at n - 1 attends."""
    return min(n, window + min(sink, max(0, n - window)))


def work(case):
    Hq, Hkv, hd = SHAPES[case["shape"]]
    row = Hkv * hd * ROW[case["kv"]]
    if case["op"] == "append":
        n = case["n_tok"]
        ids = n * 4 * (2 + len(case["axes"].split(",")) if case["axes"] else 2)
        return {"bytes": n * (2 * Hq * hd * 4 + 2 * Hkv * hd * 4 + 2 * row) + ids,
                "flops": n * (Hq + Hkv) * hd * (7 if case["norm"] else 3)}
    if case["op"] == "prefill":
        n, past = case["n_tok"], case["past"]
        pairs = sum(_seen(past + t + 1, case["window"], case["sink"]) for t in range(n))
        lo = max(0, past + 1 - case["window"])
        rows = past + n - lo + min(case["sink"], lo)
        return {"bytes": 2 * rows * row + 2 * n * Hq * hd * 4, "flops": 4 * pairs * Hq * hd}
    lens = _lens(case)
    rows = sum(_seen(n, case["window"], case["sink"]) for n in lens)
    b = 2 * rows * row + 2 * len(lens) * Hq * hd * 4
    if case["op"] == "step":
        b += len(lens) * ((Hq + 2 * Hkv) * hd * 4)
    return {"bytes": b, "flops": 4 * rows * Hq * hd}


def _tables(lens, sink, first, gen):
    """Page tables of the pages a windowed cache keeps (the others are -1), dealt in a random order.
    `first`: per sequence the first position that the call's tokens may see."""
    n_max = -(-max(lens) // PAGE)
    kept = []
    for n, lo in zip(lens, first):
        kept.append([lp for lp in range(-(-n // PAGE)) if (lp + 1) * PAGE > lo or lp * PAGE < sink])
    total = sum(map(len, kept))
    order = torch.randperm(total + 3, generator=gen, device=DEV)[:total].to(torch.int32)
    at = torch.tensor([b * n_max + lp for b, k in enumerate(kept) for lp in k], device=DEV)
    table = torch.full((len(lens) * n_max,), -1, dtype=torch.int32, device=DEV)
    table[at] = order
    return table.view(len(lens), n_max), total + 3


def _fill(pool, kv, gen):
    """Random rows in a pool of bytes."""
    if kv == "f32":
        pool.view(torch.float32).normal_(generator=gen)
    elif kv == "f16":
        pool.view(torch.float16).normal_(generator=gen)
    else:
        b = pool.view(-1, 34)
        b[:, 2:] = torch.randint(-127, 128, (b.shape[0], 32), generator=gen, device=DEV, dtype=torch.int8).view(torch.uint8)
        d = torch.rand(b.shape[0], 1, generator=gen, device=DEV) * 0.01 + 0.01
        b[:, :2] = d.to(torch.float16).view(torch.uint8)


def prepare(case, seed):
    Hq, Hkv, hd = SHAPES[case["shape"]]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    s = {"case": case, "Hq": Hq, "Hkv": Hkv, "hd": hd}
    if op in ("append", "prefill"):
        n, past = case["n_tok"], case["past"]
        s["lens"] = [past + n]
        first = [past] if op == "append" else [past + 1 - case["window"]]
        n_new = n
    else:
        s["lens"] = _lens(case)
        first = [m - case["window"] for m in s["lens"]]
        n_new = len(s["lens"])
    s["table"], n_pages = _tables(s["lens"], case.get("sink", 0), first, gen)
    page_bytes = int(PAGE * Hkv * hd * ROW[case["kv"]])
    if own:
        from strataflow_amd.paged_kv import PagedKV
        kv = s["own"] = PagedKV(1, Hq, Hkv, hd, KV_TYPE[case["kv"]], PAGE, n_pages)
        s["k"], s["v"] = kv.k[0], kv.v[0]
    else:
        s["k"], s["v"] = (torch.empty(n_pages, page_bytes, dtype=torch.uint8, device=DEV) for _ in range(2))
    _fill(s["k"], case["kv"], gen)
    _fill(s["v"], case["kv"], gen)
    if op in ("append", "step"):
        s["qkv"] = torch.randn(n_new, (Hq + 2 * Hkv) * hd, generator=gen, device=DEV)
        s["q_norm"] = 1 + 0.2 * torch.randn(hd, generator=gen, device=DEV)
        s["k_norm"] = 1 + 0.2 * torch.randn(hd, generator=gen, device=DEV)
    else:
        s["q"] = torch.randn(n_new, Hq, hd, generator=gen, device=DEV)
    if op == "append":
        s["seq"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        s["pos"] = torch.arange(past, past + n, dtype=torch.int32, device=DEV)
    elif op != "prefill":
        s["seq_len"] = torch.tensor(s["lens"], dtype=torch.int32, device=DEV)
        s["seq"] = torch.arange(n_new, dtype=torch.int32, device=DEV)
        s["pos"] = s["seq_len"] - 1
    # the rotation: a step's is the plain one of a whole head
    axes = [int(x) for x in case["axes"].split(",")] if case.get("axes") else None
    s["rot"], s["axes"], s["base"] = case.get("rot", hd), axes, 1e6
    s["neox"], s["mix"], s["norm"] = case.get("neox", True), case.get("mix", False), case.get("norm", True)
    s["rope_pos"] = None
    if axes:
        # a picture of `wide` columns after the text: time stands still, rows and columns count
        wide, off = 37, torch.arange(n, device=DEV)
        grid = [torch.full_like(off, past // 2), past // 2 + off // wide, past // 2 + off % wide]
        s["rope_pos"] = torch.stack(grid[:len(axes)]).to(torch.int32)
    if own and op in ("append", "step"):
        from strataflow_amd.paged_kv import rope_desc
        s["rope"] = rope_desc(hd, s["base"], n_rot=s["rot"], neox=s["neox"], sections=axes, interleaved=s["mix"])
    return s


# ---- the plain forms -----------------------------------------------------------------------------------

def _axis_of_pair(s):
    """The axis of each rotated pair: blocks of the sections' sizes, or dealt in turn, where an axis
    whose section is full passes its pair to the first."""
    half = s["rot"] // 2
    if not s["axes"]:
        return torch.zeros(half, dtype=torch.long, device=DEV)
    n = torch.tensor(s["axes"], device=DEV)
    i = torch.arange(half, device=DEV)
    if not s["mix"]:
        return (i[:, None] >= n.cumsum(0)[None]).sum(1)
    a, turn = i % len(s["axes"]), i // len(s["axes"])
    return torch.where(turn < n[a], a, torch.zeros_like(a))


def _turn(x, s, weight, cos, sin):
    """x [n, heads, hd] normed and rotated, in 32 bits."""
    if s["norm"]:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    r, half = s["rot"], s["rot"] // 2
    a, b = (x[..., :half], x[..., half:r]) if s["neox"] else (x[..., 0:r:2], x[..., 1:r:2])
    u, w = a * cos - b * sin, a * sin + b * cos
    y = torch.cat([u, w], -1) if s["neox"] else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _rows(pool, s):
    """A pool's rows [pages, PAGE, Hkv, ...] as they are held."""
    kv, shape = s["case"]["kv"], (-1, PAGE, s["Hkv"])
    if kv == "q8_0":
        return pool.view(*shape, s["hd"] // 32, 34)
    return pool.view(torch.float32 if kv == "f32" else torch.float16).view(*shape, s["hd"])


def _values(rows, s):
    """Rows as the 32-bit values they stand for."""
    if s["case"]["kv"] != "q8_0":
        return rows.float()
    d = rows[..., :2].contiguous().view(torch.float16).float()
    return (d * rows[..., 2:].contiguous().view(torch.int8).float()).flatten(-2)


def _held(x, s):
    """x [n, Hkv, hd] as the cache holds it."""
    if s["case"]["kv"] == "f32":
        return x
    if s["case"]["kv"] == "f16":
        return x.to(torch.float16)
    x = x.unflatten(-1, (-1, 32))
    d = x.abs().amax(-1, keepdim=True) / 127
    y = x * torch.where(d > 0, 1 / d, 0)
    y = (y.abs() + 0.5).floor() * y.sign()
    return torch.cat([d.to(torch.float16).view(torch.uint8), y.to(torch.int8).view(torch.uint8)], -1)


def _plain_append(s):
    n, Hq, Hkv, hd = s["qkv"].shape[0], s["Hq"], s["Hkv"], s["hd"]
    x = s["qkv"].view(n, Hq + 2 * Hkv, hd)
    pos = s["pos"][None] if s["rope_pos"] is None else s["rope_pos"]
    half = s["rot"] // 2
    freq = s["base"] ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    angle = pos.double()[_axis_of_pair(s)].t() * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _turn(x[:, :Hq], s, s["q_norm"], cos, sin)
    k = _turn(x[:, Hq:Hq + Hkv], s, s["k_norm"], cos, sin)
    page = s["table"][s["seq"].long(), (s["pos"] // PAGE).long()].long()
    at = (s["pos"] % PAGE).long()
    _rows(s["k"], s)[page, at] = _held(k, s)
    _rows(s["v"], s)[page, at] = _held(x[:, Hq + Hkv:], s)
    return q


def _softmax(scores):
    """Rows of -inf alone give zeros."""
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(m == -math.inf, 0, m))
    z = e.sum(-1, keepdim=True)
    return e / torch.where(z == 0, 1, z)


def _plain_decode(s, q):
    c, Hkv, hd = s["case"], s["Hkv"], s["hd"]
    B, g = q.shape[0], s["Hq"] // Hkv
    lens = s["seq_len"].long()
    lo = (lens - c["window"]).clamp(min=0)
    sinks = lo.clamp(max=c["sink"])
    j = torch.arange(max(_seen(n, c["window"], c["sink"]) for n in s["lens"]), device=DEV)
    p = torch.where(j < sinks[:, None], j, lo[:, None] + j - sinks[:, None])
    there = p < lens[:, None]
    p = torch.where(there, p, 0)
    page = s["table"].long().gather(1, p // PAGE)
    k = _values(_rows(s["k"], s)[page, p % PAGE], s).permute(0, 2, 3, 1).contiguous()
    v = _values(_rows(s["v"], s)[page, p % PAGE], s).permute(0, 2, 1, 3).contiguous()
    v = torch.where(there[:, None, :, None], v, 0)
    scores = (q.view(B, Hkv, g, hd) @ k) / math.sqrt(hd)
    scores = scores.masked_fill(~there[:, None, None], -math.inf)
    return (_softmax(scores) @ v).reshape(B, -1)


def _plain_prefill(s):
    c, Hkv, hd = s["case"], s["Hkv"], s["hd"]
    n, past, g = c["n_tok"], c["past"], s["Hq"] // Hkv
    lo = max(0, past + 1 - c["window"])
    p = torch.cat([torch.arange(min(lo, c["sink"]), device=DEV), torch.arange(lo, past + n, device=DEV)])
    page = s["table"][0].long()[p // PAGE]
    k = _values(_rows(s["k"], s)[page, p % PAGE], s).permute(1, 2, 0).contiguous()
    v = _values(_rows(s["v"], s)[page, p % PAGE], s).permute(1, 0, 2).contiguous()
    t = torch.arange(past, past + n, device=DEV)[:, None]
    sees = (p <= t) & ((p < c["sink"]) | (p > t - c["window"]))
    q = s["q"].view(n, Hkv, g, hd).permute(1, 2, 0, 3).reshape(Hkv, g * n, hd)
    scores = (q @ k) / math.sqrt(hd)
    scores = scores.view(Hkv, g, n, -1).masked_fill(~sees, -math.inf).view(Hkv, g * n, -1)
    o = _softmax(scores) @ v
    return o.view(Hkv, g, n, hd).permute(2, 0, 1, 3).reshape(n, -1)


# ---- one pass ------------------------------------------------------------------------------------------

def _own_append(s):
    n, Hq, Hkv, hd = s["qkv"].shape[0], s["Hq"], s["Hkv"], s["hd"]
    x = s["qkv"].view(n, Hq + 2 * Hkv, hd)
    return s["own"].norm_rope_append(0, x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], s["seq"], s["pos"], s["table"],
                                     s["rope"], q_norm=s["q_norm"] if s["norm"] else None,
                                     k_norm=s["k_norm"] if s["norm"] else None, eps=EPS, rope_pos=s["rope_pos"])


def run(state):
    s, c = state, state["case"]
    if c["op"] == "append":
        q = _own_append(s) if own else _plain_append(s)
        return {"q": q, "k": _rows(s["k"], s), "v": _rows(s["v"], s)}
    if c["op"] == "prefill":
        if own:
            return s["own"].prefill_window(0, s["q"], s["table"][0], c["past"], c["window"], c["sink"])
        return _plain_prefill(s)
    q = s.get("q")
    if c["op"] == "step":
        q = _own_append(s) if own else _plain_append(s)
    if own:
        out = s["own"].decode_window(0, q, s["table"], s["seq_len"], max(s["lens"]), c["window"], c["sink"])
    else:
        out = _plain_decode(s, q)
    return {"q": q, "out": out} if c["op"] == "step" else out


# ---- from the definitions, in 64 bits --------------------------------------------------------------------

def _exact_rows(pool, s):
    rows = _rows(pool, s)
    if s["case"]["kv"] != "q8_0":
        return rows.double()
    n = rows.shape[:3]
    d = rows.reshape(-1, 34)[:, :2].contiguous().view(torch.float16).double()
    return (d * rows.reshape(-1, 34)[:, 2:].contiguous().view(torch.int8).double()).view(*n, s["hd"])


def _exact_append(s):
    """(q, pool k, pool v) by complex numbers: a pair is one, a rotation a product with exp(i angle)."""
    n, Hq, Hkv, hd = s["qkv"].shape[0], s["Hq"], s["Hkv"], s["hd"]
    x = s["qkv"].double().view(n, Hq + 2 * Hkv, hd)
    r, half = s["rot"], s["rot"] // 2
    axis = []
    left = list(s["axes"] or [half])
    for i in range(half):
        if s["mix"]:
            a = i % len(left)
            a = a if a == 0 or left[a] > 0 else 0
        else:
            a = next(a for a in range(len(left)) if left[a] > 0)
        left[a] -= 1
        axis.append(a)
    assert not any(left), "sections that add up"
    pos = (s["pos"][None] if s["rope_pos"] is None else s["rope_pos"]).double()
    unit = torch.stack([torch.polar(torch.ones(n, dtype=torch.float64, device=DEV), pos[axis[i]] / s["base"] ** (i / half))
                        for i in range(half)], 1)[:, None]

    def turned(y, w):
        if s["norm"]:
            y = y / (y.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
        i = torch.arange(half, device=DEV)
        i, j = (i, i + half) if s["neox"] else (2 * i, 2 * i + 1)
        z = torch.complex(y[..., i], y[..., j]) * unit
        out = y.clone()
        out[..., i], out[..., j] = z.real, z.imag
        return out

    q, k, v = turned(x[:, :Hq], s["q_norm"]), turned(x[:, Hq:Hq + Hkv], s["k_norm"]), x[:, Hq + Hkv:]
    pk, pv = _exact_rows(s["k"], s).clone(), _exact_rows(s["v"], s).clone()
    pos, seq, table = s["pos"].tolist(), s["seq"].tolist(), s["table"].tolist()
    page = torch.tensor([table[b][p // PAGE] for b, p in zip(seq, pos)], device=DEV)
    at = torch.tensor([p % PAGE for p in pos], device=DEV)

    def held(y):
        if s["case"]["kv"] == "f16" and s["case"]["op"] == "step":
            return y.to(torch.float16).double()  # what the attention reads; a pool itself is compared unrounded
        if s["case"]["kv"] != "q8_0":
            return y
        y = y.reshape(n, Hkv, hd // 32, 32)
        d = y.abs().max(-1, keepdim=True).values / 127
        steps = torch.where(d > 0, y / d, 0)
        return (d.to(torch.float16).double() * torch.trunc(steps + 0.5 * steps.sign())).view(n, Hkv, hd)

    pk[page, at], pv[page, at] = held(k), held(v)
    return q, pk, pv


def _exact_attend(s, q, pk, pv, b, tokens, rows):
    """Row i of q [rows, Hq, hd] is the token at tokens[i] of sequence b: every position under it, by a mask."""
    c, Hkv, hd, g = s["case"], s["Hkv"], s["hd"], s["Hq"] // s["Hkv"]
    t = torch.tensor(tokens, device=DEV)[:, None]
    p = torch.arange(max(tokens) + 1, device=DEV)
    sees = (p <= t) & ((t - p < c["window"]) | (p < c["sink"]))
    p, sees = p[sees.any(0)], sees[:, sees.any(0)]
    page = s["table"][b].long()[p // PAGE]
    out = torch.zeros(rows, s["Hq"], hd, dtype=torch.float64, device=DEV)
    for h in range(s["Hq"]):
        k, v = pk[page, p % PAGE, h // g], pv[page, p % PAGE, h // g]
        w = (q[:, h].double() @ k.t().contiguous()) * hd ** -0.5
        w = torch.softmax(w.masked_fill(~sees, -math.inf), -1)
        out[:, h] = w @ v
    return out.reshape(rows, -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        q, k, v = _exact_append(s)
        return {"q": q, "k": k, "v": v}
    if case["op"] == "prefill":
        pk, pv = _exact_rows(s["k"], s), _exact_rows(s["v"], s)
        n = case["n_tok"]
        return _exact_attend(s, s["q"], pk, pv, 0, list(range(case["past"], case["past"] + n)), n)
    if case["op"] == "step":
        q, pk, pv = _exact_append(s)
    else:
        q, pk, pv = s["q"], _exact_rows(s["k"], s), _exact_rows(s["v"], s)
    out = torch.cat([_exact_attend(s, q[b:b + 1], pk, pv, b, [n - 1], 1) for b, n in enumerate(s["lens"])])
    return {"q": q, "out": out} if case["op"] == "step" else out
