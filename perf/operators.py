"""Attention under masks, attention of a batch over a shared prefix, and the cache append that feeds it, as cases
that can be timed and compared.

    own                  False: the operators in plain torch operations; True: this library's entry points
    listed()             the cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a program holds before the call: operands on the GPU and, where own, their handles
    run(state)           one pass; returns its outputs
    exact(case, seed)    the same outputs from the definition, in 64 bits
    work(case)           bytes and operations the pass cannot do without

Three kinds of case:

    masked   grouped-query attention whose rows see one range of keys each: causal, packed documents, a prefix that all
             rows of a document see; scores optionally capped by a tanh and biased by distance
    shared   the query rows of many requests against one shared prefix and each request's own (paged) cache
    append   new key and value rows normalised, rotated and put into the (paged) cache; query rows on the way
"""
from __future__ import annotations

import math

import torch

own = False

D = 128
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
CODE = {"f32": 0, "f16": 1, "bf16": 2}
ROTATION = {"none": 0, "pairs": 1, "halves": 2}
CHUNK = 1 << 28  # scores formed at a time by the plain forms


# ------------------------------------------------------------------------ cases
def masked(name, tokens, *, keys=0, batch=1, heads=32, kv=8, causal=True, docs=0, prefix=False, cap=0.0, bias=False, dtype="bf16"):
    return {"name": name, "kind": "masked", "batch": batch, "q": tokens, "k": keys or tokens, "heads": heads, "kv": kv, "causal": causal,
            "docs": docs, "prefix": prefix, "cap": cap, "bias": bias, "dtype": dtype}


def shared(name, requests, tokens, prefix, capacity, *, page=16, heads=32, kv=8, causal=True, cap=0.0, bias=False, dtype="bf16"):
    return {"name": name, "kind": "shared", "requests": requests, "q": tokens, "prefix": prefix, "capacity": capacity, "page": page,
            "heads": heads, "kv": kv, "causal": causal, "cap": cap, "bias": bias, "dtype": dtype}


def append(name, requests, tokens, capacity, *, page=16, heads=32, kv=8, act="bf16", dtype="bf16", rotation="halves", norm=True):
    return {"name": name, "kind": "append", "requests": requests, "tokens": tokens, "capacity": capacity, "page": page, "heads": heads,
            "kv": kv, "act": act, "dtype": dtype, "rotation": rotation, "norm": norm}


def listed():
    return [
        # the text encoder on one short prompt: causal, eight key heads for 32 query heads; all latency
        masked("prompt_77", 77),
        # eight prompts padded to 512 slots, real lengths from one to all of them; capped scores
        masked("prompts_padded", 512, batch=8, docs=1, cap=30.0, dtype="f16"),
        # seven renders of different sizes packed into one sequence, each attending to itself only
        masked("images_packed", 6007, heads=24, kv=24, causal=False, docs=7),
        # two sequences of a prompt that all rows see, followed by rows generated in order
        masked("prefix_rows", 4609, heads=30, kv=30, docs=2, prefix=True),
        # one very long text with a bias that falls with distance: the most work
        masked("long_bias", 16384, heads=24, kv=8, bias=True),
        # one new token of four sequences against caches of 8191 keys
        masked("one_token", 1, keys=8191, batch=4),
        # 32 requests that continue one long prompt, a token each; their own keys in pages of 16
        shared("tokens_shared_prompt", 32, 1, 4096, 320),
        # four 512 x 512 renders beside one reference image whose keys and values are kept from the first step
        shared("images_reference", 4, 1536, 4096, 1536, page=0, heads=24, kv=24, causal=False),
        # a few requests with three drafted tokens each behind a very long prompt, pages of 64, capped scores
        shared("drafts_long_prompt", 7, 3, 30011, 2000, page=64, heads=16, kv=2, cap=50.0, dtype="f16"),
        # the new token of 32 requests goes into their caches; all latency
        append("append_token", 32, 1, 320),
        # reference images of four requests enter the cache, f32 activations as the resident form keeps them
        append("append_image", 4, 4096, 4096, page=0, heads=24, kv=24, act="f32", rotation="pairs"),
        # prompts of different length, half precision, pages of 64
        append("append_prompts", 3, 1000, 1100, page=64, act="f16", dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("masked", "masked", "masked", "shared", "shared", "append"))
    heads, kv = rng.choice(((32, 8), (32, 8), (24, 24), (30, 30), (24, 8), (16, 2), (5, 5), (15, 3)))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    cap = rng.choice((0.0, 0.0, 0.0, 30.0, 50.0))
    bias = rng.random() < 0.25
    page = rng.choice((0, 8, 16, 16, 64, 256))
    if kind == "masked":
        form = rng.choice(("causal", "full", "docs", "docs", "prefix", "padded", "token", "chunk"))
        c = masked("", _log(rng, 1, 12000), heads=heads, kv=kv, cap=cap, bias=bias, dtype=dtype, causal=rng.random() < 0.6)
        if form == "causal":
            c["causal"] = True
        elif form == "docs":
            c["docs"] = min(c["q"], _log(rng, 1, 300))
        elif form == "prefix":
            c.update(docs=min(c["q"], rng.randint(1, 4)), prefix=True, causal=True)
        elif form == "padded":
            c.update(q=min(c["q"], 2000), docs=1, batch=rng.randint(2, 8), causal=True)
            c["k"] = c["q"]
        elif form == "token":
            c.update(q=rng.randint(1, 4), k=_log(rng, 4, 60000), batch=rng.randint(1, 8), causal=True)
        elif form == "chunk":
            c.update(q=min(c["q"], 3000), causal=True)
            c["k"] = c["q"] + _log(rng, 1, 12000)
    elif kind == "shared":
        if rng.random() < 0.7:
            c = shared("", _log(rng, 1, 128), rng.choice((1, 1, 1, 2, 3, 5)), _log(rng, 1, 40000), _log(rng, 8, 2000), page=page, heads=heads, kv=kv,
                       cap=cap, bias=bias, dtype=dtype)
        else:
            t = _log(rng, 16, 2000)
            c = shared("", rng.randint(1, 4), t, _log(rng, 1, 6000), t + rng.choice((0, 0, rng.randint(0, 500))), page=page, heads=heads, kv=kv,
                       causal=rng.random() < 0.5, cap=cap, bias=bias, dtype=dtype)
    else:
        t = _log(rng, 1, 3000)
        c = append("", _log(rng, 1, 64) if t < 64 else rng.randint(1, 5), t, t + rng.randint(0, 300), page=page, heads=heads, kv=kv,
                   act=rng.choice(("bf16", "f16", "f32")), dtype=dtype, rotation=rng.choice(("pairs", "halves", "halves", "none")),
                   norm=rng.random() < 0.7)
    del c["name"]
    return c


def _uneven(total, parts):
    """`parts` positive lengths, uneven, that add up to `total` (total >= parts)."""
    weight = [1 + (7 * i) % 5 + (3 * i) % 4 for i in range(parts)]
    out = [1 + (total - parts) * w // sum(weight) for w in weight]
    out[-1] += total - sum(out)
    return out


def _starts(case):
    """Document borders of each segment, or None: packed documents leave two per cent of the rows behind the last one."""
    if not case["docs"]:
        return None
    if case["batch"] > 1:  # padded segments: lengths from one row to all
        return [[0, max(1, case["q"] * (b + 1) // case["batch"])] for b in range(case["batch"])]
    used = max(case["docs"], case["q"] - case["q"] // 50)
    rows = [0]
    for n in _uneven(used, case["docs"]):
        rows.append(rows[-1] + n)
    return [rows]


def _prefixes(case):
    if not case["prefix"]:
        return None
    return [[(b - a) * (1 + i % 3) // 5 for i, (a, b) in enumerate(zip(s, s[1:]))] for s in _starts(case)]


def _own_lens(case):
    """Own keys of each request after the append: from its new rows to all of its room."""
    n, least = case["requests"], min(case["q"], case["capacity"])
    return [least + (case["capacity"] - least) * ((5 * i) % n + 1) // n for i in range(n)]


def _append_rows(case):
    """(start, count) of each request."""
    n = case["requests"]
    counts = [case["tokens"] if i % 3 == 0 else max(1, case["tokens"] * (n - i) // n) for i in range(n)]
    return [((case["capacity"] - c) * (i % 4) // 3, c) for i, c in enumerate(counts)]


def _pages(case):
    return -(-case["capacity"] // case["page"]) if case["page"] else 0


def _visible(case):
    """(query, key) pairs of one head."""
    if case["kind"] == "shared":
        pairs = 0
        for n in _own_lens(case):
            q = case["q"]
            pairs += q * case["prefix"] + (sum(max(0, t + 1 + n - q) for t in range(q)) if case["causal"] else q * n)
        return pairs
    docs = []
    starts = _starts(case)
    if starts is None:
        docs = [(case["q"], case["k"], 0)] * case["batch"]
    else:
        for b, s in enumerate(starts):
            for i, (lo, hi) in enumerate(zip(s, s[1:])):
                docs.append((hi - lo, hi - lo, _prefixes(case)[b][i] if case["prefix"] else 0))
    pairs = 0
    for q, k, p in docs:
        if not case["causal"]:
            pairs += q * k
        else:
            off = k - q
            pairs += sum(min(k, max(p, i + 1 + off, 0)) for i in range(q))
    return pairs


def work(case):
    s = SIZE[case["dtype"]]
    if case["kind"] == "append":
        rows = sum(c for _, c in _append_rows(case))
        width = (case["heads"] + 2 * case["kv"]) * D
        table = 0 if case["rotation"] == "none" else 2 * rows * D * 4
        return {"bytes": rows * width * (SIZE[case["act"]] + s) + table, "flops": rows * width * 8}
    flops = 4 * D * case["heads"] * _visible(case)
    if case["kind"] == "shared":
        keys = case["prefix"] + sum(_own_lens(case))
        rows = case["requests"] * case["q"]
    else:
        starts = _starts(case)
        rows = case["batch"] * case["q"] if starts is None else sum(x[-1] for x in starts)
        keys = case["batch"] * case["k"] if starts is None else rows
    return {"bytes": (2 * rows * case["heads"] + 2 * keys * case["kv"]) * D * s, "flops": flops}


# ---------------------------------------------------------------------- operands
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, scale=1.0):
    """In pieces, so that the f32 draws of a large operand are never all there at once."""
    out = torch.empty(shape, device="cuda", dtype=TORCH[dtype])
    flat = out.view(-1)
    for a in range(0, flat.numel(), 1 << 27):
        b = min(flat.numel(), a + (1 << 27))
        flat[a:b] = (torch.randn(b - a, generator=g, device="cuda") * scale).to(TORCH[dtype])
    return out


def _u32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda", dtype=torch.float32)


def _table(requests, pages, g):
    """Pages of the requests, scattered over a pool with a few spare ones."""
    pool = requests * pages + 3
    order = torch.randperm(pool, generator=g, device="cuda")
    return order[: requests * pages].to(torch.int32).view(requests, pages).contiguous(), pool


def _inputs(case, seed):
    g = _generator(seed)
    dt, heads, kv = case["dtype"], case["heads"], case["kv"]
    s = {"case": case}
    if case["kind"] == "masked":
        b = case["batch"]
        s["q"] = _randn(g, (b, case["q"], heads, D), dt, 1.2)
        s["k"] = _randn(g, (b, case["k"], kv, D), dt)
        s["v"] = _randn(g, (b, case["k"], kv, D), dt)
        s["out"] = torch.zeros_like(s["q"])
        if case["docs"]:
            s["starts"] = _u32(_starts(case))
        if case["prefix"]:
            s["prefix"] = _u32(_prefixes(case))
        if case["bias"]:
            s["slopes"] = _slopes(heads)
    elif case["kind"] == "shared":
        n = case["requests"]
        s["q"] = _randn(g, (n, case["q"], heads, D), dt, 1.2)
        s["pk"] = _randn(g, (case["prefix"], kv, D), dt)
        s["pv"] = _randn(g, (case["prefix"], kv, D), dt)
        if case["page"]:
            s["table"], pool = _table(n, _pages(case), g)
            shape = (pool, case["page"], kv, D)
        else:
            shape = (n, case["capacity"], kv, D)
        s["k"] = _randn(g, shape, dt)
        s["v"] = _randn(g, shape, dt)
        s["out"] = torch.zeros_like(s["q"])
        s["lens"] = _u32(_own_lens(case))
        if case["bias"]:
            s["slopes"] = _slopes(heads)
    else:
        n, t = case["requests"], case["tokens"]
        s["q"] = _randn(g, (n, t, heads, D), case["act"], 2.0)
        s["k"] = _randn(g, (n, t, kv, D), case["act"], 2.0)
        s["v"] = _randn(g, (n, t, kv, D), case["act"])
        if case["page"]:
            s["table"], pool = _table(n, _pages(case), g)
            shape = (pool, case["page"], kv, D)
        else:
            shape = (n, case["capacity"], kv, D)
        s["ck"] = torch.zeros(shape, device="cuda", dtype=TORCH[dt])
        s["cv"] = torch.zeros_like(s["ck"])
        s["qo"] = torch.zeros((n, t, heads, D), device="cuda", dtype=TORCH[dt])
        s["begin"] = _u32([a for a, _ in _append_rows(case)])
        s["count"] = _u32([c for _, c in _append_rows(case)])
        if case["norm"]:
            s["wq"] = 1.0 + 0.1 * torch.randn(D, generator=g, device="cuda")
            s["wk"] = 1.0 + 0.1 * torch.randn(D, generator=g, device="cuda")
        if case["rotation"] != "none":
            pos = torch.arange(case["capacity"], device="cuda", dtype=torch.float64)
            freq = 10000.0 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))
            ang = pos[:, None] * freq[None, :]
            ang = ang.repeat_interleave(2, 1) if case["rotation"] == "pairs" else torch.cat((ang, ang), 1)
            s["cos"], s["sin"] = ang.cos().float().contiguous(), ang.sin().float().contiguous()
    return s


EPS = 1e-6


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _bind(s)
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _call(s)
    return {"masked": _plain_masked, "shared": _plain_shared, "append": _plain_append}[kind](s)


# ------------------------------------------------------------------- plain forms
def _attend(q, k, v, seen, cap, slopes, gap):
    """q [rows][heads][D], k and v [keys][kv][D], in f32: softmax(cap(q k^T / sqrt(D)) - slope gap) v over the keys that
    seen(rows) -> [rows][keys] admits; zeros for a row that sees none. gap(rows) -> [rows][keys] is the distance."""
    rows, heads, _ = q.shape
    keys, kv, _ = k.shape
    group = heads // kv
    if keys == 0:
        return torch.zeros_like(q)
    qt = q.view(rows, kv, group, D).permute(1, 2, 0, 3).contiguous()  # [kv][group][rows][D]
    kt = k.permute(1, 2, 0).contiguous()                              # [kv][D][keys]
    vt = v.permute(1, 0, 2).contiguous()                              # [kv][keys][D]
    out = torch.empty_like(qt)
    step = max(1, min(rows, CHUNK // (keys * group)))
    heads_at_once = max(1, min(kv, CHUNK // (keys * group * step)))
    sl = None if slopes is None else slopes.view(kv, group, 1, 1)
    for a in range(0, rows, step):
        n = min(step, rows - a)
        ids = torch.arange(a, a + n, device=q.device)
        mask = seen(ids)
        far = None if slopes is None else gap(ids).float()
        for h in range(0, kv, heads_at_once):
            e = min(kv, h + heads_at_once)
            x = torch.bmm(qt[h:e, :, a:a + n].reshape(e - h, group * n, D), kt[h:e]).view(e - h, group, n, keys)
            x *= 1.0 / math.sqrt(D)
            if cap:
                x = cap * torch.tanh(x / cap)
            if far is not None:
                x = x - sl[h:e] * far
            if mask is not None:
                x.masked_fill_(~mask, -math.inf)
            top = x.amax(-1, keepdim=True)
            x = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = x.sum(-1, keepdim=True)
            y = torch.bmm(x.view(e - h, group * n, keys), vt[h:e]).view(e - h, group, n, D)
            out[h:e, :, a:a + n] = torch.where(total > 0, y / total, torch.zeros_like(y))
    return out.permute(2, 0, 1, 3).reshape(rows, heads, D)


def _plain_masked(s):
    c = s["case"]
    starts, prefixes = _starts(c), _prefixes(c)
    for b in range(c["batch"]):
        borders = starts[b] if starts else None
        spans = [(0, c["q"], 0, c["k"], 0)] if borders is None else [
            (x, y, x, y, prefixes[b][i] if prefixes else 0) for i, (x, y) in enumerate(zip(borders, borders[1:]))]
        for q0, q1, k0, k1, p in spans:
            nk, off = k1 - k0, (k1 - k0) - (q1 - q0)
            j = torch.arange(nk, device="cuda")
            seen = (lambda i: (j[None, :] <= i[:, None] + off) | (j[None, :] < p)) if c["causal"] else (lambda i: None)
            gap = lambda i: (i[:, None] + off - j[None, :]).abs()
            y = _attend(s["q"][b, q0:q1].float(), s["k"][b, k0:k1].float(), s["v"][b, k0:k1].float(), seen, c["cap"], s.get("slopes"), gap)
            s["out"][b, q0:q1] = y.to(s["out"].dtype)
    return s["out"]


def _own_rows(s, name):
    """A request's own keys or values, [requests][capacity][kv][D]."""
    c = s["case"]
    if not c["page"]:
        return s[name]
    x = s[name][s["table"].long()]
    return x.flatten(1, 2)[:, : c["capacity"]]


def _plain_shared(s):
    """The scores of all requests against the prefix as one product, those against their own keys as one batch."""
    c = s["case"]
    n, t, heads, kv, p, cap = c["requests"], c["q"], c["heads"], c["kv"], c["prefix"], c["capacity"]
    group = heads // kv
    q = s["q"].float().view(n, t, kv, group, D).permute(2, 0, 3, 1, 4).contiguous()  # [kv][n][group][t][D]
    pk, pv = s["pk"].float().permute(1, 2, 0).contiguous(), s["pv"].float().permute(1, 0, 2).contiguous()
    ok = _own_rows(s, "k").float().permute(2, 0, 3, 1).contiguous()  # [kv][n][D][cap]
    ov = _own_rows(s, "v").float().permute(2, 0, 1, 3).contiguous()  # [kv][n][cap][D]
    lens = s["lens"].view(n, 1, 1, 1)
    row = torch.arange(t, device="cuda").view(1, 1, t, 1)
    j = torch.arange(cap, device="cuda").view(1, 1, 1, cap)
    mask = j < lens
    if c["causal"]:
        mask = mask & (j <= row + lens - t)
    far_p = far_o = None
    if c["bias"]:
        at = (p + lens - t + row).float()
        far_p = (at - torch.arange(p, device="cuda").view(1, 1, 1, p)).abs()
        far_o = (at - (p + j)).abs()
    out = s["out"].view(n, t, kv, group, D)
    step = max(1, min(n, CHUNK // (group * t * (p + cap))))
    for h in range(kv):
        for a in range(0, n, step):
            e = min(n, a + step)
            x = torch.cat((torch.mm(q[h, a:e].reshape(-1, D), pk[h]).view(e - a, group, t, p),
                           torch.bmm(q[h, a:e].reshape(e - a, group * t, D), ok[h, a:e]).view(e - a, group, t, cap)), -1)
            x *= 1.0 / math.sqrt(D)
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if c["bias"]:
                x = x - s["slopes"].view(kv, 1, group, 1, 1)[h] * torch.cat((far_p[a:e], far_o[a:e]), -1)
            x[..., p:].masked_fill_(~mask[a:e], -math.inf)
            x = torch.exp(x - x.amax(-1, keepdim=True))
            total = x.sum(-1, keepdim=True)
            y = torch.mm(x[..., :p].reshape(-1, p), pv[h]).view(e - a, group, t, D)
            y = y + torch.bmm(x[..., p:].reshape(e - a, group * t, cap), ov[h, a:e]).view(e - a, group, t, D)
            out[a:e, :, h] = (y / total).permute(0, 2, 1, 3).to(out.dtype)
    return s["out"]


def _plain_append(s):
    c = s["case"]
    n, t = c["requests"], c["tokens"]
    tok = torch.arange(t, device="cuda").view(1, t)
    row = s["begin"].long().view(n, 1) + tok
    live = tok < s["count"].view(n, 1)
    at = torch.where(live, row, torch.zeros_like(row))

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        if c["rotation"] == "none":
            return x
        cos, sin = s["cos"][at].unsqueeze(2), s["sin"][at].unsqueeze(2)
        if c["rotation"] == "pairs":
            other = torch.stack((-x[..., 1::2], x[..., 0::2]), -1).flatten(-2)
        else:
            other = torch.cat((-x[..., D // 2:], x[..., : D // 2]), -1)
        return x * cos + other * sin

    q, k, v = turned(s["q"], s.get("wq")), turned(s["k"], s.get("wk")), s["v"].float()
    s["qo"][live] = q[live].to(s["qo"].dtype)
    req = torch.arange(n, device="cuda").view(n, 1).expand(n, t)[live]
    pos = row[live]
    if c["page"]:
        where = (s["table"].long()[req, pos // c["page"]], pos % c["page"])
    else:
        where = (req, pos)
    s["ck"].index_put_(where, k[live].to(s["ck"].dtype))
    s["cv"].index_put_(where, v[live].to(s["cv"].dtype))
    return {"q": s["qo"], "k": s["ck"], "v": s["cv"]}


# --------------------------------------------------------------------- definition
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, s)
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    heads, group = case["heads"], case["heads"] // case["kv"]

    def rows(q, k, v, visible, position, key_position):
        """One head at a time: q [rows][D]; visible [rows] counts of leading keys in f64 order, or None for all."""
        step = max(1, (1 << 27) // max(1, k.shape[0]))
        y = torch.zeros((q.shape[0], heads, D), device="cuda", dtype=torch.float64)
        for h in range(heads):
            kh, vh = k[:, h // group].double().t().contiguous(), v[:, h // group].double()
            for a in range(0, q.shape[0], step):
                qq = q[a:a + step, h].double()
                x = qq @ kh / math.sqrt(D)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["bias"]:
                    x = x - s["slopes"][h].double() * (position[a:a + step, None] - key_position[None, :]).abs().double()
                if visible is not None:
                    x = torch.where(torch.arange(k.shape[0], device="cuda")[None, :] < visible[a:a + step, None], x, torch.full_like(x, -math.inf))
                y[a:a + step, h] = torch.nan_to_num(torch.softmax(x, -1), nan=0.0) @ vh
        return y

    if case["kind"] == "masked":
        starts, prefixes = _starts(case), _prefixes(case)
        for b in range(case["batch"]):
            docs = [(0, case["q"], 0, case["k"], 0)] if starts is None else []
            if starts is not None:
                for i in range(len(starts[b]) - 1):
                    lo, hi = starts[b][i], starts[b][i + 1]
                    docs.append((lo, hi, lo, hi, prefixes[b][i] if prefixes else 0))
            for q0, q1, k0, k1, p in docs:
                i = torch.arange(q1 - q0, device="cuda") + (k1 - k0) - (q1 - q0)
                visible = (i + 1).clamp(min=p) if case["causal"] else None
                out[b, q0:q1] = rows(s["q"][b, q0:q1], s["k"][b, k0:k1], s["v"][b, k0:k1], visible, i, torch.arange(k1 - k0, device="cuda"))
        return out
    for b, n in enumerate(_own_lens(case)):
        parts = []
        for name in ("k", "v"):
            x = s[name][b] if not case["page"] else torch.cat([s[name][i] for i in s["table"][b].tolist()])
            parts.append(torch.cat((s["p" + name], x[:n])))
        i = torch.arange(case["q"], device="cuda") + case["prefix"] + n - case["q"]
        out[b] = rows(s["q"][b], parts[0], parts[1], i + 1 if case["causal"] else None, i, torch.arange(case["prefix"] + n, device="cuda"))
    return out


def _exact_append(case, s):
    f64 = lambda t: t.double()
    q = torch.zeros(s["qo"].shape, device="cuda", dtype=torch.float64)
    k = torch.zeros(s["ck"].shape, device="cuda", dtype=torch.float64)
    v = torch.zeros_like(k)

    def turned(x, w, first):
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * f64(w)
        if case["rotation"] == "none":
            return x
        c, d = f64(s["cos"][first:first + x.shape[0]])[:, None], f64(s["sin"][first:first + x.shape[0]])[:, None]
        y = torch.empty_like(x)
        a, b = (slice(0, D, 2), slice(1, D, 2)) if case["rotation"] == "pairs" else (slice(0, D // 2), slice(D // 2, D))
        y[..., a] = x[..., a] * c[..., a] - x[..., b] * d[..., a]
        y[..., b] = x[..., b] * c[..., b] + x[..., a] * d[..., b]
        return y

    for r, (first, count) in enumerate(_append_rows(case)):
        q[r, :count] = turned(f64(s["q"][r, :count]), s.get("wq"), first)
        kk, vv = turned(f64(s["k"][r, :count]), s.get("wk"), first), f64(s["v"][r, :count])
        if not case["page"]:
            k[r, first:first + count], v[r, first:first + count] = kk, vv
            continue
        pos = torch.arange(first, first + count, device="cuda")
        page, slot = s["table"][r].long()[pos // case["page"]], pos % case["page"]
        k[page, slot], v[page, slot] = kk, vv
    return {"q": q, "k": k, "v": v}


# -------------------------------------------------------------- this library's calls
_ctx = None


def _context():
    """One context per process: device, queue, pipelines."""
    global _ctx
    if _ctx is None:
        from zdraw_amd import host

        torch.zeros(1, device="cuda")  # torch's runtime first: both then use the same device context
        _ctx = host.Context.init()
    return _ctx


class _Wrapped:
    """A tensor in GPU memory that the library sees through a handle."""

    def __init__(self, t):
        from zdraw_amd import hip

        self.t, self.lib = t, hip.lib()
        self.handle = self.lib.zdraw_hip_wrap_device_memory(_context().device, t.data_ptr(), t.numel() * t.element_size())
        if not self.handle:
            raise RuntimeError(hip.last_error())

    def __del__(self):
        if getattr(self, "handle", None):
            self.lib.zdraw_hip_release_buffer(self.handle)
            self.handle = None


def _dense(dst, t):
    """Strides of [a][b][c][D] in elements."""
    for i in range(3):
        dst[i] = t.stride(i)


def _bind(s):
    """Handles and argument structs, which a program keeps from call to call."""
    from zdraw_amd import hip

    c = s["case"]
    w = {name: _Wrapped(t) for name, t in s.items() if torch.is_tensor(t)}
    h = lambda name: w[name].handle if name in w else None
    if c["kind"] == "masked":
        p, o = hip.MaskedAttn(), hip.MaskOperands()
        p.batch, p.q_tokens, p.k_tokens = c["batch"], c["q"], c["k"]
        p.causal, p.documents, p.softcap = int(c["causal"]), c["docs"], c["cap"]
        for name, dst in (("q", p.q_stride), ("k", p.k_stride), ("v", p.v_stride), ("out", p.out_stride)):
            _dense(dst, s[name])
        o.q_starts, o.prefix, o.slopes = h("starts"), h("prefix"), h("slopes")
        s["args"] = (h("q"), h("k"), h("v"), h("out"))
        s["fn"] = "zdraw_hip_run_attention_masked"
    elif c["kind"] == "shared":
        p, o = hip.SharedAttn(), hip.SharedOperands()
        p.requests, p.q_tokens, p.prefix_tokens, p.capacity = c["requests"], c["q"], c["prefix"], c["capacity"]
        p.page_tokens, p.pages = c["page"], s["k"].shape[0] if c["page"] else 0
        p.causal, p.softcap = int(c["causal"]), c["cap"]
        for name, dst in (("q", p.q_stride), ("out", p.out_stride), ("k", p.k_stride), ("v", p.v_stride)):
            _dense(dst, s[name])
        for name, dst in (("pk", p.prefix_k_stride), ("pv", p.prefix_v_stride)):
            dst[0], dst[1] = s[name].stride(0), s[name].stride(1)
        o.lens, o.page_table, o.slopes = h("lens"), h("table"), h("slopes")
        s["args"] = (h("q"), h("pk"), h("pv"), h("k"), h("v"), h("out"))
        s["fn"] = "zdraw_hip_run_attention_shared"
    else:
        p, o = hip.KvAppend(), hip.AppendOperands()
        p.requests, p.tokens, p.capacity = c["requests"], c["tokens"], c["capacity"]
        p.page_tokens, p.pages = c["page"], s["ck"].shape[0] if c["page"] else 0
        p.in_dtype, p.rotation, p.eps = CODE[c["act"]], ROTATION[c["rotation"]], EPS
        p.rope_rows = s["cos"].shape[0] if "cos" in s else 0
        for name, dst in (("q", p.q_stride), ("k", p.k_stride), ("v", p.v_stride), ("qo", p.q_out_stride), ("ck", p.cache_k_stride),
                          ("cv", p.cache_v_stride)):
            _dense(dst, s[name])
        o.starts, o.counts, o.page_table = h("begin"), h("count"), h("table")
        o.q_weight, o.k_weight, o.rope_cos, o.rope_sin = h("wq"), h("wk"), h("cos"), h("sin")
        s["args"] = (h("q"), h("k"), h("v"), h("qo"), h("ck"), h("cv"))
        s["fn"] = "zdraw_hip_run_kv_append"
    p.heads, p.kv_heads, p.head_dim, p.dtype = c["heads"], c["kv"], D, CODE[c["dtype"]]
    s["params"], s["ops"], s["wrapped"] = p, o, w


def _call(s):
    import ctypes

    from zdraw_amd import hip

    rc = getattr(hip.lib(), s["fn"])(_context().queue, *s["args"], ctypes.byref(s["params"]), ctypes.byref(s["ops"]))
    if rc != 0:
        raise RuntimeError(f"{s['fn']} rc={rc}: {hip.last_error()}")
    return s["out"] if s["case"]["kind"] != "append" else {"q": s["qo"], "k": s["ck"], "v": s["cv"]}
