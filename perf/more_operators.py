"""Measured cases of a step that checks trees of drafted tokens: its projections, its attention, what it keeps.

A drafted step gives each request a tree of tokens behind its cached rows.  The model runs once over all of them;
the longest path whose tokens the model itself would have produced is kept.  Five operators are measured:

- gemm:   FP8 E4M3 weights with a UE8M0 scale per 128 x 128 times the step's tokens, quantised per block of a row;
- tree:   from each token's parent, the bits of its ancestors and its position;
- attend: softmax attention of the tree's queries over the paged 4-bit cache, each over the cached rows and its ancestors;
- accept: the path that agrees with the model's own tokens, the new lengths, and the blocks that go back on the stack;
- commit: the kept rows moved to their places in the cache; they come back as the values that they stand for.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
# rows, cols of a weight
WEIGHTS = {
    "wq_a": (1024, 4096),   # DeepSeek-V4's attention projections
    "wq_b": (32768, 1024),
    "wkv": (512, 4096),
    "wo_b": (4096, 8192),
    "w1": (2048, 4096),     # its shared expert's
    "w2": (4096, 2048),
    "square": (4096, 4096),  # the GEMV benchmark's
    "odd": (1000, 1360),    # neither a multiple of the block
}
# heads, kv heads, head_dim, whether values have a cache of their own
LAYOUTS = {
    "latent": (64, 1, 512, False),   # DeepSeek-V4's attention: 64 heads over one shared 512-wide row
    "grouped": (32, 8, 128, True),   # 4 query heads to a kv head
    "odd": (28, 4, 128, True),       # 7 query heads to a kv head
    "narrow": (64, 8, 64, True),     # 64-wide heads
    "wide": (16, 2, 256, True),      # 256-wide heads
    "single": (8, 8, 128, True),     # every head has its own rows
}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
VOCAB = 129280


def listed():
    return [
        # one token of one user: latency, and the weight's bytes
        _gemm("gemm-square-1-f32", "square", 1, "f32", 64),
        # a full server's drafted step: 32 requests of up to 16 tokens
        _gemm("gemm-wo_b-509-bf16", "wo_b", 509, "bf16", 128),
        # a long prompt, in the model path's own type: operations
        _gemm("gemm-wo_b-8192-f32", "wo_b", 8192, "f32", 64),
        # a server's step: masks and positions of small trees
        _tree("tree-32x16", 32, 16),
        # many requests, wide trees
        _tree("tree-1000x100", 1000, 100),
        # one user, one small tree, a short context: latency
        _attend("attend-latent-1x97x8-f32", "latent", 1, 97, 8, "f32", sink=True),
        # a full server at the decode benchmark's position, 16 drafted tokens a request
        _attend("attend-latent-32x4096x16-bf16", "latent", 32, 4096, 16, "bf16", sink=True),
        # grouped heads, an odd group, larger trees, ragged pages
        _attend("attend-odd-24x2999x33-bf16", "odd", 24, 2999, 33, "bf16", page=48),
        # the server's step: what is kept, which blocks go back
        _accept("accept-32x16", 32, 16, 4096, 64),
        # many requests with wide trees over small pages
        _accept("accept-1000x100", 1000, 100, 2048, 16),
        # one latent layer of a few requests
        _commit("commit-latent-8x8", "latent", 1, 8, 8, 64),
        # every layer of the model at once (layers lie inside a block), a full server
        _commit("commit-latent-43-32x16", "latent", 43, 32, 16, 64),
    ]


def _gemm(name, weight, tokens, dtype, block):
    return {"name": name, "op": "gemm", "weight": weight, "tokens": tokens, "dtype": dtype, "block": block}


def _tree(name, requests, nodes):
    return {"name": name, "op": "tree", "requests": requests, "nodes": nodes}


def _attend(name, layout, requests, length, nodes, dtype, page=64, window=0, first=0, sink=False):
    return {"name": name, "op": "attend", "layout": layout, "requests": requests, "length": length, "nodes": nodes, "dtype": dtype,
            "page": page, "window": window, "first": first, "sink": sink}


def _accept(name, requests, nodes, length, page):
    return {"name": name, "op": "accept", "requests": requests, "nodes": nodes, "length": length, "page": page}


def _commit(name, layout, layers, requests, nodes, page):
    return {"name": name, "op": "commit", "layout": layout, "layers": layers, "requests": requests, "nodes": nodes, "page": page}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.random()
    if kind < 0.35:
        weight = rng.choice(sorted(WEIGHTS))
        most = min(8192, 8192 * sum(WEIGHTS["wo_b"]) // sum(WEIGHTS[weight]))  # within the largest listed one's bytes
        c = _gemm("", weight, _log(rng, 1, most), rng.choice(sorted(DTYPES)), rng.choice((32, 64, 128)))
    elif kind < 0.45:
        c = _tree("", _log(rng, 1, 1000), _log(rng, 1, 100))
    elif kind < 0.8:
        layout = rng.choice(("latent", "latent") + tuple(sorted(LAYOUTS)))
        requests, nodes = _log(rng, 1, 48), _log(rng, 2, 64)
        # a drawn pass stays within the largest listed one's operations
        heads, _, d, _ = LAYOUTS[layout]
        most = min(16384, (32 * 16 * 4096 * 64 * 512) // (requests * nodes * heads * d))
        window = rng.choice((0, 0, 0, 128, 1000))
        c = _attend("", layout, requests, _log(rng, min(most, 2 * nodes), max(most, 2 * nodes)), nodes, rng.choice(sorted(DTYPES)),
                    page=rng.choice((16, 48, 64, 128)), window=window, first=rng.choice((0, 4, 70)) if window else 0,
                    sink=rng.random() < 0.5)
    elif kind < 0.9:
        c = _accept("", _log(rng, 1, 1000), _log(rng, 1, 100), _log(rng, 1, 4096), rng.choice((16, 48, 64)))
    else:
        layout = rng.choice(("latent",) + tuple(sorted(LAYOUTS)))
        c = _commit("", layout, rng.choice((1, 2, 5, 43) if layout == "latent" else (1, 2, 5)), _log(rng, 1, 32), _log(rng, 3, 64),
                    rng.choice((16, 24, 64)))
    c.pop("name")
    return c


# ---------------------------------------------------------------------------
# lengths: a function of the case alone
# ---------------------------------------------------------------------------
def _nodes(case):
    """Tokens of each request's tree; the first one has the most."""
    n = case["nodes"]
    return [n if i == 0 else 1 + (i * 7 + 3) % n for i in range(case["requests"])]


def _lengths(case):
    """(kv length, tree tokens) of each request; the first one has the full length, the others spread below it."""
    out = []
    for i, n in enumerate(_nodes(case)):
        part = 1.0 if i == 0 else 0.25 + 0.75 * ((i * 0.6180339887) % 1.0)
        out.append((max(n, int(round(case["length"] * part))), n))
    return out


def _touched(case, base):
    """Cached rows that at least one query of the tree sees: the root's window reaches back farthest."""
    if not case["window"]:
        return base
    start = max(0, base + 1 - case["window"])
    return base - start + min(case["first"], start)


def _keep(nodes):
    """Tokens kept in the commit cases: about a third."""
    return [1 + (n - 1) // 3 for n in nodes]


def work(case):
    op = case["op"]
    if op == "gemm":
        rows, cols = WEIGHTS[case["weight"]]
        t, size = case["tokens"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": rows * cols + -(-rows // 128) * -(-cols // 128) + t * (rows + cols) * size, "flops": 2 * t * rows * cols}
    if op == "tree":
        t, words = sum(_nodes(case)), -(-case["nodes"] // 64)
        return {"bytes": t * (4 + 8 * words + 4) + case["requests"] * 8, "flops": 0}
    if op == "accept":
        t = sum(_nodes(case))
        return {"bytes": t * (3 * 4 + 4) + case["requests"] * 5 * 4, "flops": 0}
    heads, kvh, d, sep = LAYOUTS[case["layout"]]
    row = kvh * (d // 2 + d // 32) * (2 if sep else 1)
    if op == "commit":
        nodes = _nodes(case)
        moved = sum(k - 1 for k in _keep(nodes)) * case["layers"]
        wide = kvh * d * (2 if sep else 1)
        return {"bytes": 2 * moved * row + sum(nodes) * case["layers"] * (row + 2 * wide), "flops": 0}
    size = 4 if case["dtype"] == "f32" else 2
    bytes_, flops = 0, 0
    for n, q in _lengths(case):
        seen = _touched(case, n - q)
        bytes_ += (seen + q) * row + 2 * q * heads * d * size + q * 16 + 8 + 4 * -(-n // case["page"])
        # a node has about log2 of the tree's size ancestors; the cached rows are nearly all of it
        flops += 4 * heads * d * q * (seen + 1)
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _parents(rng, nodes):
    """Drafts as they are grown: a token continues one of the last few, often the last.  Indices inside the request; -1: the root."""
    out = []
    for n in nodes:
        j = np.arange(n)
        back = np.minimum(rng.integers(0, 4, n) * (rng.random(n) < 0.6), np.maximum(j - 1, 0))
        p = j - 1 - back
        p[:1] = -1
        out.append(p)
    return np.concatenate(out).astype(np.int32)


def _int32(x):
    return torch.tensor(np.asarray(x, np.int32), device=DEV)


def _starts(counts):
    return [0] + [int(x) for x in np.cumsum(counts)]


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


def _table(g, pages, blocks):
    """Block table of requests that hold `pages` blocks each of a shuffled pool, and the blocks that are left."""
    order = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(pages), max(pages)), -1, dtype=torch.int32, device=DEV)
    cols = torch.arange(max(pages), device=DEV)
    table[cols[None, :] < torch.tensor(pages, device=DEV)[:, None]] = order[:sum(pages)]
    return table, order[sum(pages):]


def prepare(case, seed):
    g, rng = _generator(seed), np.random.default_rng(seed)
    op = case["op"]
    if op == "gemm":
        rows, cols = WEIGHTS[case["weight"]]
        # trained weights: about unit codes of E4M3 (saturated, never its NaN), block scales over a few octaves
        w = (torch.randn(rows, cols, generator=g, device=DEV) * 40).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        scale = torch.randint(112, 119, (-(-rows // 128), -(-cols // 128)), generator=g, device=DEV).to(torch.uint8)
        x = _rows(g, case["tokens"], 1, cols).squeeze(1).to(DTYPES[case["dtype"]])
        return {"case": case, "w": w, "scale": scale, "x": x}
    nodes = _nodes(case)
    starts = _starts(nodes)
    s = {"case": case, "starts": _int32(starts), "tokens": starts[-1]}
    if op == "tree":
        s["parents"] = _int32(_parents(rng, nodes))
        s["lens"] = _int32(rng.integers(0, 4096, len(nodes)) + np.array(nodes))
        return s
    if op == "accept":
        parents = _parents(rng, nodes)
        # drafts from a small model's favourites; most nodes have a child that the large model agrees with
        drafts = rng.integers(0, 50, starts[-1]) * 1931 % VOCAB
        targets = rng.integers(0, VOCAB, starts[-1])
        at = np.repeat(np.array(starts[:-1]), nodes)
        agree = np.flatnonzero((parents >= 0) & (rng.random(starts[-1]) < 0.6))
        targets[at[agree] + parents[agree]] = drafts[agree]
        page, lens = case["page"], [n for n, _ in _lengths(case)]
        pages = [-(-n // page) for n in lens]
        table, left = _table(g, pages, sum(pages) + 9)
        free = torch.full((sum(pages) + 9,), -1, dtype=torch.int32, device=DEV)
        free[:9] = left
        s.update(parents=_int32(parents), drafts=_int32(drafts), targets=_int32(targets), lens=_int32(lens), table=table, free=free,
                 top=_int32([9]))
        return s
    heads, kvh, d, sep = LAYOUTS[case["layout"]]
    page = case["page"]
    if op == "commit":
        lens = [n + (i * 389 + 17) % 1000 for i, n in enumerate(nodes)]
        pages = [-(-n // page) for n in lens]
        kvh *= case["layers"]
        keep = _keep(nodes)
        path = np.full(starts[-1], -1, np.int32)
        for r, (n, k) in enumerate(zip(nodes, keep)):
            # a path late in the tree's order (so that a second pass moves the same rows to the same places)
            path[starts[r]:starts[r] + k] = np.concatenate(([0], k + np.sort(rng.permutation(n - k)[:k - 1])))
        blocks = sum(pages) + 3
        k, ks = _pool(g, blocks, kvh, page, d)
        v, vs = _pool(g, blocks, kvh, page, d) if sep else (None, None)
        table, _ = _table(g, pages, blocks)
        who = np.repeat(np.arange(len(nodes)), nodes)
        pos = np.array(lens)[who] - np.array(nodes)[who] + np.arange(starts[-1]) - np.array(starts)[who]
        every = table[torch.tensor(who, device=DEV), torch.tensor(pos // page, device=DEV)].long() * page + torch.tensor(pos % page, device=DEV)
        s.update(k=k, ks=ks, v=v, vs=vs, table=table, lens=_int32(lens), path=_int32(path), counts=_int32(keep), every=every, most=max(keep))
        return s
    lens = _lengths(case)
    pages = [-(-n // page) for n, _ in lens]
    blocks = sum(pages) + 3
    k, ks = _pool(g, blocks, kvh, page, d)
    v, vs = _pool(g, blocks, kvh, page, d) if sep else (None, None)
    table, _ = _table(g, pages, blocks)
    # scores with a spread of about 1.5, as a trained layer's
    queries = (torch.randn(starts[-1], heads, d, generator=g, device=DEV) * 1.5).to(DTYPES[case["dtype"]])
    s.update(k=k, ks=ks, v=v, vs=vs, table=table, q=queries, parents=_int32(_parents(rng, nodes)), lens=_int32([n for n, _ in lens]),
             max_len=max(n for n, _ in lens), sink=torch.randn(heads, generator=g, device=DEV) if case["sink"] else None)
    s["masks"], s["positions"] = _plain_tree(s)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _e4m3(t):
    """The nearest E4M3 value of |t| <= 448, ties to the lower one."""
    a = t.abs()
    # spacing of the grid at a: 2^(e - 3), 2^-9 below 2^-6
    e = torch.clamp((a.view(torch.int32) >> 23) - 127, min=-6)
    step = ((e - 3 + 127) << 23).view(torch.float32)
    y = a / step
    low = torch.floor(y)
    rest = y - low
    up = (rest > 0.5) | ((rest == 0.5) & (t < 0))
    return torch.where(t < 0, -1.0, 1.0) * (low + up) * step


def _act_quant(x, block):
    """x [t, c] as the product takes it: per `block` columns the least 2^k with max(amax, 1e-4) <= 448 * 2^k, then E4M3."""
    t, c = x.shape
    pad = -c % block
    b = torch.cat((x.float(), torch.zeros(t, pad, device=x.device)), 1).view(t, -1, block)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True).clamp(min=1e-4))
    k = torch.where(m <= 0.875, e - 9, e - 8)
    scale = ((k + 127) << 23).view(torch.float32)
    return (_e4m3((b / scale).clamp(-448, 448)) * scale).view(t, -1)[:, :c]


def _e4m3_values(w):
    """Bytes -> values (no NaN among them)."""
    mag = ((w & 127).int() << 20).view(torch.float32) * 2.0 ** 120
    return torch.where(w >= 128, -mag, mag)


def _plain_gemm(s):
    w = _e4m3_values(s["w"])
    scale = (s["scale"].int() << 23).view(torch.float32)
    scale = scale.repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :w.shape[1]]
    return torch.matmul(_act_quant(s["x"], s["case"]["block"]), (w * scale).t()).to(s["x"].dtype)


def _owner(s):
    """Request of each token, and its index there."""
    t = torch.arange(s["tokens"], device=DEV)
    starts = s["starts"].long()
    who = torch.searchsorted(starts, t, right=True) - 1
    return who, t - starts[who]


def _plain_tree(s):
    who, j = _owner(s)
    first = s["starts"].long()[who]
    words = -(-s["case"]["nodes"] // 64)
    # bit by bit of the request's tokens; a token's ancestors are found by doubling the steps taken
    sees = torch.arange(64 * words, device=DEV)[None, :] == j[:, None]
    up = s["parents"].long()
    depth = (up >= 0).long()
    for _ in range(max(1, (s["case"]["nodes"] - 1).bit_length())):
        live = up >= 0
        at = torch.where(live, first + up, first)
        sees = sees | (sees[at] & live[:, None])
        depth = depth + torch.where(live, depth[at], torch.zeros_like(depth))
        up = torch.where(live, up[at], up)
    bits = sees.view(-1, words, 64).long() << torch.arange(64, device=DEV)
    counts = s["starts"][1:] - s["starts"][:-1]
    return bits.sum(-1), (s["lens"][who] - counts[who] + depth).int()


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


_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _values(codes, scales):
    """codes [..., d/2], scales [..., d/32] -> [..., d] f32."""
    table = torch.tensor(_MAGNITUDES + tuple(-m for m in _MAGNITUDES), device=codes.device)
    x = table[torch.stack((codes & 15, codes >> 4), -1).int()].flatten(-2)
    s = (scales.int() << 23).view(torch.float32)
    return (x.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _plain_attend(s):
    case, q, lens, starts = s["case"], s["q"], s["lens"].long(), s["starts"].long()
    heads, kvh, d, _ = LAYOUTS[case["layout"]]
    b, nq, window, first, page = case["requests"], case["nodes"], case["window"], case["first"], case["page"]
    base = lens - (starts[1:] - starts[:-1])
    # rows that some query of the request may see: the first ones, then from the window's reach on
    if window and first + window + nq < s["max_len"]:
        tail = base[:, None] + 1 - window + torch.arange(window - 1 + nq, device=DEV)
        tail = torch.where(tail >= first, tail, torch.full_like(tail, -1))
        at = torch.cat((torch.arange(first, device=DEV).expand(b, -1), tail), 1)
    else:
        at = torch.arange(s["max_len"], device=DEV).expand(b, -1)
    real = (at >= 0) & (at < lens[:, None])
    where = at.clamp(min=0)
    block = torch.gather(s["table"].long(), 1, (where // page).clamp(max=s["table"].shape[1] - 1))
    block, row = torch.where(real, block, torch.zeros_like(block)), where % page

    def rows(codes, scales):
        x = _values(codes[block, :, row], scales[block, :, row])  # [b, l, kvh, d]
        return torch.where(real[:, :, None, None], x, torch.zeros_like(x)).transpose(1, 2)

    k = rows(s["k"], s["ks"])
    v = k if s["v"] is None else rows(s["v"], s["vs"])
    token = (starts[:-1, None] + torch.arange(nq, device=DEV)).clamp(max=q.shape[0] - 1)
    x = q[token].float().view(b, nq, kvh, heads // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, kvh, -1, d)
    score = (torch.matmul(x, k.transpose(2, 3)) * (d ** -0.5)).view(b, kvh, nq, heads // kvh, -1)
    pos = s["positions"].long()[token]
    rel = at - base[:, None]  # place among the tree's rows
    word = s["masks"][token]  # [b, nq, words]
    pick = torch.gather(word, 2, (rel // 64).clamp(0, word.shape[2] - 1)[:, None, :].expand(-1, nq, -1))
    own_row = (rel >= 0)[:, None, :] & ((pick >> (rel % 64)[:, None, :]) & 1).bool()
    old_row = (rel < 0)[:, None, :].expand(-1, nq, -1)
    if window:
        old_row = old_row & ((at[:, None, :] > pos[:, :, None] - window) | (at[:, None, :] < first))
    seen = real[:, None, :] & (own_row | old_row)
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
    who, j = _owner(s)
    return o[who, j].to(q.dtype)


def _plain_accept(s):
    page, n = s["case"]["page"], s["case"]["nodes"]
    starts, lens = s["starts"].long(), s["lens"].long()
    counts = starts[1:] - starts[:-1]
    j = torch.arange(n, device=DEV)
    there = j < counts[:, None]
    token = (starts[:-1, None] + j).clamp(max=s["tokens"] - 1)
    parent = torch.where(there, s["parents"][token].long(), torch.full_like(token, -2))
    draft, target = s["drafts"][token], s["targets"][token]
    at = torch.zeros_like(counts)
    alive = counts > 0
    path = [torch.where(alive, at, torch.full_like(at, -1))]
    for _ in range(1, n):
        fits = alive[:, None] & (parent == at[:, None]) & (draft == torch.gather(target, 1, at[:, None]))
        child = torch.where(fits, j, torch.full_like(token, n)).amin(1)
        alive = child < n
        at = torch.where(alive, child, at)
        path.append(torch.where(alive, child, torch.full_like(child, -1)))
    path = torch.stack(path, 1)
    kept = (path >= 0).sum(1)
    after = lens - counts + kept
    held, need = (lens + page - 1) // page, (after + page - 1) // page
    gone = held - need
    free, top = s["free"].clone(), s["top"].long()
    col = torch.arange(s["table"].shape[1], device=DEV)[None, :]
    goes = (col >= need[:, None]) & (col < held[:, None])
    to = top + torch.cumsum(gone, 0)[:, None] - gone[:, None] + col - need[:, None]
    grown = torch.cat((free, free.new_zeros(1)))
    grown[torch.where(goes, to, torch.full_like(to, free.numel()))] = s["table"]
    who, i = _owner(s)
    return {"counts": kept.int(), "path": path[who, i].int(), "next": torch.gather(target, 1, at[:, None])[:, 0], "lens": after.int(),
            "free": grown[:-1], "top": (top + gone.sum()).int()}


def _plain_commit(s):
    page, starts, lens = s["case"]["page"], s["starts"].long(), s["lens"].long()
    base = lens - (starts[1:] - starts[:-1])
    i = torch.arange(s["most"], device=DEV)
    kept = i < s["counts"][:, None]
    path = s["path"][(starts[:-1, None] + i).clamp(max=s["tokens"] - 1)].long()
    src = base[:, None] + torch.where(kept, path, torch.zeros_like(path))
    dst = base[:, None] + torch.where(kept, i, torch.zeros_like(path))
    b0, b1 = (torch.gather(s["table"].long(), 1, x // page) for x in (src, dst))
    out = []
    for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        if codes is not None:
            for x in (codes, scales):
                x[b1, :, dst % page] = x[b0, :, src % page]
            e = s["every"]
            out.append(_values(codes[e // page, :, e % page], scales[e // page, :, e % page]).to(torch.bfloat16))
    return out


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
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        return {"gemm": _plain_gemm, "tree": _plain_tree, "attend": _plain_attend, "accept": _plain_accept, "commit": _plain_commit}[op](s)
    W, ctx = _framework()
    if op == "gemm":
        return W.gemm_fp8_e4m3_ue8m0(ctx, s["w"], s["scale"], s["x"], act_quant_block=case["block"])
    if op == "tree":
        t = W.kv_tree(ctx, s["parents"], s["starts"], s["lens"], case["nodes"])
        return t.masks, t.positions
    if op == "accept":
        a = W.kv_accept(ctx, case["page"], s["parents"], s["drafts"], s["targets"], s["starts"], s["lens"], s["table"], s["free"], s["top"])
        return {"counts": a.counts, "path": a.path, "next": a.next_tokens, "lens": a.kv_lens, "free": s["free"], "top": a.free_top}
    cache = W.PagedKvCache(s["k"], s["ks"], s["v"], s["vs"])
    if op == "commit":
        W.kv_commit(ctx, cache, s["counts"], s["path"], s["starts"], s["lens"], s["table"])
        k, v = W.kv_gather(ctx, cache, s["every"], torch.bfloat16)
        return [k] if v is None else [k, v]
    return W.kv_tree_attention(ctx, cache, s["q"], s["starts"], s["lens"], s["table"], W.KvTree(s["masks"], s["positions"]),
                               window=case["window"], first=case["first"], sink=s["sink"])


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _real(codes, scales):
    c = torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()
    e, m = (c % 8) // 2, (c % 2).double()
    x = torch.where(e > 0, (1 + m / 2) * 2.0 ** (e - 1).double(), m / 2) * (1.0 - 2.0 * (c // 8).double())
    s = scales.double()
    return (x.unflatten(-1, (-1, 32)) * torch.where(s > 0, 2.0 ** (s - 127), torch.zeros_like(s))[..., None]).flatten(-2)


def _exact_gemm(s):
    block = s["case"]["block"]
    w = s["w"].long()
    e, m = (w % 128) // 8, (w % 8).double()
    real = torch.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7).double(), m / 8 * 2.0 ** -6) * (1.0 - 2.0 * (w // 128).double())
    for i in range(s["scale"].shape[0]):
        for j in range(s["scale"].shape[1]):
            real[128 * i:128 * i + 128, 128 * j:128 * j + 128] *= 2.0 ** (int(s["scale"][i, j]) - 127)
    grid = torch.tensor(sorted({(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)} | {m * 2.0 ** -9 for m in range(8)}),
                        dtype=torch.float64, device=DEV)
    grid = grid[grid <= 448]
    grid = torch.cat((-grid.flip(0)[:-1], grid))
    x = s["x"].double()
    for c in range(0, x.shape[1], block):
        part = x[:, c:c + block]
        k = torch.ceil(torch.log2(part.abs().amax(1, keepdim=True).clamp(min=1e-4) / 448))
        y = part / 2.0 ** k
        up = torch.searchsorted(grid, y.contiguous()).clamp(1, grid.numel() - 1)
        low, high = grid[up - 1], grid[up]
        x[:, c:c + block] = torch.where(y > (low + high) / 2, high, low) * 2.0 ** k
    return x @ real.t()


def exact(case, seed):
    if case["op"] in ("tree", "accept"):
        return None
    s = prepare(case, seed)
    if case["op"] == "gemm":
        return _exact_gemm(s)
    heads, kvh, d, sep = LAYOUTS[case["layout"]]
    starts, lens, page = s["starts"].tolist(), s["lens"].tolist(), case["page"]
    if case["op"] == "commit":
        out = []
        path, keep, table = s["path"].tolist(), s["counts"].tolist(), s["table"].tolist()
        src, dst = [], []
        for r, k in enumerate(keep):
            base = lens[r] - (starts[r + 1] - starts[r])
            for i in range(k):
                a, b = base + path[starts[r] + i], base + i
                src.append(table[r][a // page] * page + a % page)
                dst.append(table[r][b // page] * page + b % page)
        src, dst = (torch.tensor(x, device=DEV) for x in (src, dst))
        for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            if codes is not None:
                c, x = (t.transpose(1, 2).flatten(0, 1) for t in (codes, scales))
                c, x = c.clone(), x.clone()
                c[dst], x[dst] = c[src], x[src]
                out.append(_real(c[s["every"]], x[s["every"]]))
        return out
    got = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    parents = s["parents"].tolist()
    for r, n in enumerate(lens):
        t0, t1 = starts[r], starts[r + 1]
        base = n - (t1 - t0)
        i = torch.arange(n, device=DEV)
        block, row = s["table"][r].long()[i // page], i % page
        k = _real(s["k"][block, :, row], s["ks"][block, :, row])
        v = _real(s["v"][block, :, row], s["vs"][block, :, row]) if sep else k
        for t in range(t0, t1):
            line, up = [], t - t0
            while up >= 0:
                line.append(up)
                up = parents[t0 + up]
            p = base + len(line) - 1
            see = i < base
            if case["window"]:
                see &= (i >= p + 1 - case["window"]) | (i < case["first"])
            see[[base + x for x in line]] = True
            at = torch.nonzero(see).flatten()
            x = s["q"][t].double().view(kvh, heads // kvh, d)
            w = torch.einsum("hgd,lhd->hgl", x, k[at]) / math.sqrt(d)
            if s["sink"] is not None:
                w = torch.cat((w, s["sink"].double().view(kvh, -1, 1)), -1)
            w = torch.softmax(w, -1)[..., :at.numel()]
            got[t] = torch.einsum("hgl,lhd->hgd", w, v[at]).reshape(heads, d)
    return got
