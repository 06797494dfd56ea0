"""Measured cases of the paged 4-bit key/value cache: its plan, its writes and reads, its attention.

A cache is a pool of blocks of `page` rows per kv head; a row holds head_dim E2M1
codes (two a byte, low nibble = even column) and one UE8M0 scale per 32 of them.
Three operators are measured:

- plan:   block tables, slot maps, positions and lengths of one serving step, from
          the requests' lengths and a stack of free blocks;
- append: new rows quantised into their slots; the pool's rows come back as the
          values they stand for, read by the gather that exists for that;
- attend: softmax attention of ragged queries over the cached rows, with an optional
          sliding window, first tokens that stay visible, and a sink logit per head.
"""
import math

import torch

own = False

DEV = "cuda"
# heads, kv heads, head_dim, whether values have a cache of their own
LAYOUTS = {
    "latent": (64, 1, 512, False),   # DeepSeek-V4's attention: 64 heads over one shared 512-wide row
    "grouped": (32, 8, 128, True),   # 4 query heads to a kv head
    "odd": (28, 4, 128, True),       # 7 query heads to a kv head
    "narrow": (64, 8, 64, True),     # 64-wide heads
    "wide": (16, 2, 256, True),      # 256-wide heads
    "single": (8, 8, 128, True),     # every head has its own rows
}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one user, one token, a short context: latency
        _attend("attend-latent-1x97-f32", "latent", 1, 97, "f32", sink=True),
        # the decode benchmark's batch and position, in the model path's own type
        _attend("attend-latent-32x4096-f32", "latent", 32, 4096, "f32", sink=True),
        # a full server, twice the position, 16-bit activations
        _attend("attend-latent-32x8192-bf16", "latent", 32, 8192, "bf16", sink=True),
        # one long document (the YaRN original length): the rows are split over the GPU
        _attend("attend-latent-1x65536-bf16", "latent", 1, 65536, "bf16"),
        # a sliding-window layer far into long contexts, with first tokens kept
        _attend("attend-window-32x32768-f32", "latent", 32, 32768, "f32", window=128, first=4, sink=True),
        # grouped heads, ragged long contexts: bandwidth
        _attend("attend-grouped-16x16384-bf16", "grouped", 16, 16384, "bf16", page=16),
        # several tokens a request (a checked draft): causal inside the step, odd group and sizes
        _attend("attend-odd-24x2999-bf16", "odd", 24, 2999, "bf16", q=5, page=48),
        # one decode step's new rows
        _append("append-latent-32-f32", "latent", 32, "f32", blocks=48, page=64),
        # a prompt's rows, keys and values
        _append("append-grouped-8191-bf16", "grouped", 8191, "bf16", blocks=600, page=16),
        # the decode batch's step
        _plan("plan-32-decode", 32, 4096, 1, 64, 0),
        # a mixed step: prompts among decodes, some requests ending
        _plan("plan-1000-mixed", 1000, 2048, 96, 16, 17),
    ]


def _attend(name, layout, requests, length, dtype, q=1, page=64, window=0, first=0, sink=False):
    return {"name": name, "op": "attend", "layout": layout, "requests": requests, "length": length, "dtype": dtype,
            "q": q, "page": page, "window": window, "first": first, "sink": sink}


def _append(name, layout, rows, dtype, blocks, page):
    return {"name": name, "op": "append", "layout": layout, "rows": rows, "dtype": dtype, "blocks": blocks, "page": page}


def _plan(name, requests, length, q, page, ending):
    return {"name": name, "op": "plan", "requests": requests, "length": length, "q": q, "page": page, "ending": ending}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.random()
    if kind < 0.2:
        c = _plan("", _log(rng, 1, 1000), _log(rng, 8, 4096), rng.choice((1, 1, 3, 33, 96)), rng.choice((16, 48, 64)),
                  rng.choice((0, 5, 17)))
    elif kind < 0.4:
        rows, page = _log(rng, 1, 8191), rng.choice((16, 24, 64))
        c = _append("", rng.choice(sorted(LAYOUTS)), rows, rng.choice(sorted(DTYPES)), -(-rows // page) + rng.randint(1, 64), page)
    else:
        layout = rng.choice(("latent", "latent", "latent") + tuple(sorted(LAYOUTS)))
        q = rng.choice((1, 1, 1, 1, 2, 3, 5, 8))
        requests = _log(rng, 1, 64)
        # a drawn pass stays within the largest listed one (262144 latent rows)
        most = min(65536, 262144 // requests // (2 if q > 1 else 1))
        window = rng.choice((0, 0, 0, 128, 1000))
        c = _attend("", layout, requests, _log(rng, 1, most // 2 if layout != "latent" else most), rng.choice(sorted(DTYPES)),
                    q=q, page=rng.choice((16, 48, 64, 128)), window=window, first=rng.choice((0, 4, 70)) if window else 0,
                    sink=rng.random() < 0.5)
    c.pop("name")
    return c


# ---------------------------------------------------------------------------
# lengths: a function of the case alone
# ---------------------------------------------------------------------------
def _lengths(case):
    """(kv length, query length) of each request; the first one has the full length, the others spread below it."""
    out = []
    for i in range(case["requests"]):
        q = 1 + (i * 7 + 3) % case["q"] if case["q"] > 1 else 1
        part = 1.0 if i == 0 else 0.25 + 0.75 * ((i * 0.6180339887) % 1.0)
        out.append((max(q, int(round(case["length"] * part))), q))
    return out


def _visible(case, n, t):
    """How many rows a query at position t of a request with n rows sees."""
    last = t + 1
    if not case["window"]:
        return last
    start = max(0, last - case["window"])
    return last - start + min(case["first"], start)


def _touched(case, n, q):
    """How many rows at least one of the request's q queries sees."""
    if not case["window"]:
        return n
    start = max(0, n - q + 1 - case["window"])
    return n - start + min(case["first"], start)


def work(case):
    if case["op"] == "plan":
        old, new, ending = _plan_lengths(case)
        page = case["page"]
        tokens = sum(new)
        fresh = sum(-(-(o + n) // page) - -(-o // page) for o, n, e in zip(old, new, ending) if not e)
        freed = sum(-(-o // page) for o, e in zip(old, ending) if e)
        return {"bytes": case["requests"] * (4 + 4 + 1 + 4 + 4) + (fresh + freed) * 8 + tokens * 16, "flops": 0}
    heads, kvh, d, sep = LAYOUTS[case["layout"]]
    size = 4 if case["dtype"] == "f32" else 2
    row = kvh * (d // 2 + d // 32) * (2 if sep else 1)
    if case["op"] == "append":
        read = case["blocks"] * case["page"]
        wide = kvh * d * (2 if sep else 1)
        return {"bytes": case["rows"] * (wide * size + row + 8) + read * (row + wide * 2), "flops": 0}
    bytes_, flops = 0, 0
    for n, q in _lengths(case):
        bytes_ += _touched(case, n, q) * row + 2 * q * heads * d * size + 8 + 4 * -(-n // case["page"])
        flops += sum(4 * heads * d * _visible(case, n, n - q + j) for j in range(q))
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _rows(g, rows, kvh, d):
    """Normed key/value rows: unit variance, a few channels several times larger, as trained norms leave them."""
    gain = 1.0 + 4.0 * (torch.rand(kvh, d, generator=g, device=DEV) < 0.02)
    return torch.randn(rows, kvh, d, generator=g, device=DEV) * gain


def _pool(g, blocks, kvh, page, d):
    """A pool that earlier steps filled: codes [blocks, kvh, page, d/2], scales [blocks, kvh, page, d/32]."""
    codes = torch.empty(blocks, kvh, page, d // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(blocks, kvh, page, d // 32, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 25) // (kvh * page * d))
    for b in range(0, blocks, step):
        n = min(step, blocks - b)
        c, s = _quantise(_rows(g, n * page, kvh, d))
        codes[b:b + n] = c.view(n, page, kvh, d // 2).transpose(1, 2)
        scales[b:b + n] = s.view(n, page, kvh, d // 32).transpose(1, 2)
    return codes, scales


def _plan_lengths(case):
    old, new, ending = [], [], []
    for i in range(case["requests"]):
        e = case["ending"] > 0 and i % case["ending"] == case["ending"] - 1
        o = 0 if i % 5 == 4 else (i * 389 + 17) % case["length"]
        old.append(o)
        new.append(0 if e else 1 if i % 3 else 1 + (i * 31) % case["q"])
        ending.append(e)
    return old, new, ending


def _shuffled(g, n):
    return torch.randperm(n, generator=g, device=DEV).to(torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "plan":
        old, new, ending = _plan_lengths(case)
        page = case["page"]
        held = [-(-o // page) for o in old]
        most = max(-(-(o + n) // page) for o, n in zip(old, new)) + 1
        fresh = sum(-(-(o + n) // page) for o, n in zip(old, new)) - sum(held)
        blocks = sum(held) + fresh + 9
        order = _shuffled(g, blocks)
        table = torch.full((case["requests"], most), -1, dtype=torch.int32, device=DEV)
        cols = torch.arange(most, device=DEV)
        table[cols[None, :] < torch.tensor(held, device=DEV)[:, None]] = order[:sum(held)]
        free = torch.full((blocks,), -1, dtype=torch.int32, device=DEV)
        free[:blocks - sum(held)] = order[sum(held):]
        return {"case": case, "table": table, "free": free,
                "top": torch.tensor([blocks - sum(held)], dtype=torch.int32, device=DEV),
                "old": torch.tensor(old, dtype=torch.int32, device=DEV), "new": torch.tensor(new, dtype=torch.int32, device=DEV),
                "ending": torch.tensor(ending, dtype=torch.uint8, device=DEV), "tokens": sum(new)}
    heads, kvh, d, sep = LAYOUTS[case["layout"]]
    page, dtype = case["page"], DTYPES[case["dtype"]]
    if case["op"] == "append":
        k, ks = _pool(g, case["blocks"], kvh, page, d)
        v, vs = _pool(g, case["blocks"], kvh, page, d) if sep else (None, None)
        total = case["blocks"] * page
        s = {"case": case, "k": k, "ks": ks, "v": v, "vs": vs, "every": torch.arange(total, device=DEV),
             "slots": torch.randperm(total, generator=g, device=DEV)[:case["rows"]].clone(),
             "new_k": _rows(g, case["rows"], kvh, d).to(dtype), "new_v": _rows(g, case["rows"], kvh, d).to(dtype) if sep else None}
        return s
    lens = _lengths(case)
    pages = [-(-n // page) for n, _ in lens]
    blocks = sum(pages) + 3
    k, ks = _pool(g, blocks, kvh, page, d)
    v, vs = _pool(g, blocks, kvh, page, d) if sep else (None, None)
    table = torch.full((case["requests"], max(pages)), -1, dtype=torch.int32, device=DEV)
    order = _shuffled(g, blocks)
    cols = torch.arange(max(pages), device=DEV)
    table[cols[None, :] < torch.tensor(pages, device=DEV)[:, None]] = order[:sum(pages)]
    starts = [0]
    for _, q in lens:
        starts.append(starts[-1] + q)
    # scores with a spread of about 1.5, as a trained layer's
    queries = (torch.randn(starts[-1], heads, d, generator=g, device=DEV) * 1.5).to(dtype)
    return {"case": case, "k": k, "ks": ks, "v": v, "vs": vs, "table": table, "q": queries,
            "starts": torch.tensor(starts, dtype=torch.int32, device=DEV), "lens": torch.tensor([n for n, _ in lens], dtype=torch.int32, device=DEV),
            "max_len": max(n for n, _ in lens), "max_q": max(q for _, q in lens),
            "sink": torch.randn(heads, generator=g, device=DEV) if case["sink"] else None}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantise(x):
    """x [..., d] -> codes [..., d/2], scales [..., d/32]: the smallest power of two (at least 2^-126, at most 2^125)
    whose 6-fold holds the block's largest value, each value to the nearest code, ties to the even one."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1)
    bits = top.view(torch.int32)
    k = (bits >> 23) - 127 - 2 + ((bits & 0x7FFFFF) > 0x400000).int()
    k = torch.clamp(k, -126, 125)
    a = b.abs() * ((127 - k) << 23).view(torch.float32)[..., None]
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)) | (torch.signbit(b).to(torch.uint8) << 3)
    code = code.reshape(*x.shape[:-1], -1, 2)
    scale = torch.where(top > 0, k + 127, torch.zeros_like(k)).to(torch.uint8)
    return code[..., 0] | (code[..., 1] << 4), scale


def _values(codes, scales):
    """codes [..., d/2], scales [..., d/32] -> [..., d] f32."""
    table = torch.tensor(_MAGNITUDES + tuple(-m for m in _MAGNITUDES), device=codes.device)
    x = table[torch.stack((codes & 15, codes >> 4), -1).int()].flatten(-2)
    s = (scales.int() << 23).view(torch.float32)
    return (x.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _plain_plan(s):
    page = s["case"]["page"]
    old, new, ending, top = s["old"].long(), s["new"].long(), s["ending"].bool(), s["top"].long()
    table, free = s["table"].clone(), s["free"].clone()
    held = (old + page - 1) // page
    after = torch.where(ending, torch.zeros_like(old), old + new)
    fresh = torch.where(ending, torch.zeros_like(old), (after + page - 1) // page - held)
    freed = torch.where(ending, held, torch.zeros_like(held))
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    # blocks of ending requests go on the stack, in the order of requests and pages
    gone = ending[:, None] & (col < held[:, None])
    to = top + torch.cumsum(freed, 0)[:, None] - freed[:, None] + col
    grown = torch.cat((free, free.new_zeros(1)))
    grown[torch.where(gone, to, torch.full_like(to, free.numel()))] = table
    free = grown[:-1]
    top = top + freed.sum()
    # new pages come off its top in the same order
    due = (col >= held[:, None]) & (col < (held + fresh)[:, None])
    at = top - 1 - (torch.cumsum(fresh, 0)[:, None] - fresh[:, None] + col - held[:, None])
    table = torch.where(due, free[at.clamp(0, free.numel() - 1)], table)
    starts = torch.cat((new.new_zeros(1), torch.cumsum(new, 0)))
    t = torch.arange(s["tokens"], device=table.device)
    who = torch.searchsorted(starts, t, right=True) - 1
    pos = old[who] + t - starts[who]
    slots = table[who, pos // page].long() * page + pos % page
    return {"table": table, "free": free, "top": (top - fresh.sum()).int(), "lens": after.int(), "starts": starts.int(),
            "slots": slots, "positions": pos.int(), "requests": who.int()}


def _plain_append(s):
    page = s["case"]["page"]
    out = []
    for codes, scales, rows in ((s["k"], s["ks"], s["new_k"]), (s["v"], s["vs"], s["new_v"])):
        if codes is not None:
            c, x = _quantise(rows)
            codes[s["slots"] // page, :, s["slots"] % page] = c
            scales[s["slots"] // page, :, s["slots"] % page] = x
            out.append(_values(codes, scales).transpose(1, 2).reshape(-1, codes.shape[1], 2 * codes.shape[3]).to(torch.bfloat16))
    return out


def _plain_attend(s):
    case, q, lens, starts = s["case"], s["q"], s["lens"].long(), s["starts"].long()
    heads, kvh, d, _ = LAYOUTS[case["layout"]]
    b, nq, window, first = case["requests"], s["max_q"], case["window"], case["first"]
    counts = starts[1:] - starts[:-1]
    # the rows that any query of the request may see
    if window and first + window + nq - 1 < s["max_len"]:
        tail = lens[:, None] - (window + nq - 1) + torch.arange(window + nq - 1, device=q.device)
        tail = torch.where(tail >= first, tail, torch.full_like(tail, -1))
        head = torch.arange(first, device=q.device).expand(b, -1)
        at = torch.cat((head, tail), 1)
    else:
        at = torch.arange(s["max_len"], device=q.device).expand(b, -1)
    real = (at >= 0) & (at < lens[:, None])
    where = at.clamp(min=0)
    block = torch.gather(s["table"].long(), 1, (where // case["page"]).clamp(max=s["table"].shape[1] - 1))
    block, row = torch.where(real, block, torch.zeros_like(block)), where % case["page"]

    def rows(codes, scales):
        x = _values(codes[block, :, row], scales[block, :, row])  # [b, l, kvh, d]
        return torch.where(real[:, :, None, None], x, torch.zeros_like(x)).transpose(1, 2)

    k = rows(s["k"], s["ks"])
    v = k if s["v"] is None else rows(s["v"], s["vs"])
    j = torch.arange(nq, device=q.device)
    token = (starts[:-1, None] + j).clamp(max=q.shape[0] - 1)
    x = q[token].float().view(b, nq, kvh, heads // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, kvh, -1, d)
    score = (torch.matmul(x, k.transpose(2, 3)) * (d ** -0.5)).view(b, kvh, nq, heads // kvh, -1)
    pos = lens[:, None] - counts[:, None] + j
    seen = real[:, None, :] & (at[:, None, :] <= pos[:, :, None])
    if window:
        seen = seen & ((at[:, None, :] > pos[:, :, None] - window) | (at[:, None, :] < first))
    score = torch.where(seen[:, None, :, None, :], score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    sink = None if s["sink"] is None else s["sink"].view(1, kvh, 1, heads // kvh, 1)
    top = top if sink is None else torch.maximum(top, sink)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    total = total if sink is None else total + torch.exp(sink - top)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p.view(b, kvh, -1, p.shape[-1]), v).view(b, kvh, nq, heads // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, nq, heads, d)
    t = torch.arange(q.shape[0], device=q.device)
    who = torch.searchsorted(starts, t, right=True) - 1
    return o[who, t - starts[who]].to(q.dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
_kept = {}


def _framework():
    """The package and the process's context, which a program creates once."""
    if not _kept:
        import wohper_b200 as W

        _kept["it"] = (W, W.Context(torch.cuda.current_device()))
    return _kept["it"]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[op](state)
    W, ctx = _framework()
    if op == "plan":
        p = W.kv_plan(ctx, state["case"]["page"], state["old"], state["new"], state["table"], state["free"], state["top"],
                      state["tokens"], finished=state["ending"])
        return {"table": state["table"], "free": state["free"], "top": p.free_top, "lens": p.kv_lens, "starts": p.cu_q,
                "slots": p.slots, "positions": p.positions, "requests": p.requests}
    cache = W.PagedKvCache(state["k"], state["ks"], state["v"], state["vs"])
    if op == "append":
        W.kv_append(ctx, cache, state["slots"], state["new_k"], state["new_v"])
        k, v = W.kv_gather(ctx, cache, state["every"], torch.bfloat16)
        return [k] if v is None else [k, v]
    return W.kv_attention(ctx, cache, state["q"], state["starts"], state["lens"], state["table"], window=state["case"]["window"],
                          first=state["case"]["first"], sink=state["sink"])


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _real(codes, scales):
    c = torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()
    e, m = (c % 8) // 2, (c % 2).double()
    x = torch.where(e > 0, (1 + m / 2) * 2.0 ** (e - 1).double(), m / 2) * (1.0 - 2.0 * (c // 8).double())
    s = scales.double()
    return (x.unflatten(-1, (-1, 32)) * torch.where(s > 0, 2.0 ** (s - 127), torch.zeros_like(s))[..., None]).flatten(-2)


def _rounded(x):
    """Rows as the cache holds them: per 32 the least 2^k with 6 * 2^k >= max, the nearest of the code's values, ties to an even code."""
    x = x.double().unflatten(-1, (-1, 32))
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    unit = 2.0 ** torch.where(m <= 0.75, e - 3, e - 2).double()
    grid = torch.tensor(_MAGNITUDES, dtype=torch.float64, device=x.device)
    y = x.abs() / unit
    up = torch.searchsorted(grid, y.contiguous()).clamp(1, 7)
    low, high = grid[up - 1], grid[up]
    mid = (low + high) / 2
    near = torch.where((y > mid) | ((y == mid) & (up % 2 == 0)), high, low)
    return (torch.sign(x) * near * unit).flatten(-2)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    heads, kvh, d, sep = LAYOUTS[case["layout"]]
    if case["op"] == "append":
        out = []
        for codes, scales, rows in ((s["k"], s["ks"], s["new_k"]), (s["v"], s["vs"], s["new_v"])):
            if codes is not None:
                x = _real(codes, scales).permute(0, 2, 1, 3).reshape(-1, kvh, d)
                x[s["slots"]] = _rounded(rows)
                out.append(x)
        return out
    got = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    t = 0
    for r, (n, nq) in enumerate(_lengths(case)):
        i = torch.arange(n, device=DEV)
        block, row = s["table"][r].long()[i // case["page"]], i % case["page"]
        k = _real(s["k"][block, :, row], s["ks"][block, :, row])
        v = _real(s["v"][block, :, row], s["vs"][block, :, row]) if sep else k
        for j in range(nq):
            p = n - nq + j
            see = i <= p
            if case["window"]:
                see &= (i >= p + 1 - case["window"]) | (i < case["first"])
            at = torch.nonzero(see).flatten()
            x = s["q"][t].double().view(kvh, heads // kvh, d)
            w = torch.einsum("hgd,lhd->hgl", x, k[at]) / math.sqrt(d)
            if s["sink"] is not None:
                w = torch.cat((w, s["sink"].double().view(kvh, -1, 1)), -1)
            w = torch.softmax(w, -1)[..., :at.numel()]
            got[t] = torch.einsum("hgl,lhd->hgd", w, v[at]).reshape(heads, d)
            t += 1
    return got
