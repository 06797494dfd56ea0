"""Trees of drafted tokens over the paged 4-bit cache on the GPU: masks and positions,
attention, accepted paths and moved rows, against plain forms (tests/tree_reference.py).

Masks, positions, paths, lengths, stacks and moved bytes are whole numbers and equal.
The attention's tolerances are kv_attention's (tests/test_gpu_kvcache.py, from the
same sums): per output element, V and S the largest |value| and |score| the query sees,
V 2^-22 (16 + 8 S) for f32; for 16-bit queries V 2^-11 more for weights of 11 bits,
and the output's rounding, 2^-8 (bf16) or 2^-11 (f16) of it, 2^-25 for f16's subnormals.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import kv_reference as R
from tests import tree_reference as T

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 0.0, BF16: 2.0**-8, F16: 2.0**-11}
I32 = np.int32


@pytest.fixture(scope="module")
def W():
    import wohper_b200

    wohper_b200.lib()
    return wohper_b200


@pytest.fixture(scope="module")
def ctx(W):
    c = W.Context(0)
    yield c
    c.close()


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def starts(nodes):
    return np.concatenate([[0], np.cumsum(nodes)]).astype(I32)


def raises(W, ctx, kind="DeviceArg"):
    with pytest.raises(W.WohperError) as e:
        ctx.sync()
    assert e.value.kind == kind


# ---------------------------------------------------------------------------
# masks and positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("nodes", [[1], [5, 0, 64, 1, 33], [64] * 40, [65, 128, 3], [256, 0, 200, 129]], ids=str)
@pytest.mark.parametrize("chain", [0.0, 0.5, 1.0])
def test_tree(ctx, W, nodes, chain):
    rng = np.random.default_rng(sum(nodes))
    cu, most = starts(nodes), max(nodes)
    parents, spare = T.grow(rng, nodes, chain), 7  # a fixed token count larger than the step's
    lens = [n + int(rng.integers(0, 5000)) for n in nodes]
    tokens = int(cu[-1]) + spare
    t = W.kv_tree(ctx, dev(np.concatenate([parents, np.full(spare, 99, I32)])), dev(cu), dev(np.array(lens, I32)), most)
    ctx.sync()
    masks, pos = T.tree(parents, cu, lens, tokens, -(-most // 64))
    np.testing.assert_array_equal(t.masks.cpu().numpy(), masks)
    np.testing.assert_array_equal(t.positions.cpu().numpy(), pos)


def test_tree_of_many_requests(ctx, W):
    rng = np.random.default_rng(1)
    nodes = rng.integers(0, 9, 5000).tolist()
    cu, parents = starts(nodes), T.grow(rng, nodes)
    lens = [n + int(rng.integers(0, 100)) for n in nodes]
    t = W.kv_tree(ctx, dev(parents), dev(cu), dev(np.array(lens, I32)), 8)
    masks, pos = T.tree(parents, cu, lens, int(cu[-1]), 1)
    np.testing.assert_array_equal(t.masks.cpu().numpy(), masks)
    np.testing.assert_array_equal(t.positions.cpu().numpy(), pos)
    ctx.sync()


@pytest.mark.parametrize("bad", [-2, 3, 4, 1000, -2**31])
def test_tree_bad_parents_are_roots_and_recorded(ctx, W, bad):
    parents = np.array([-1, 0, 1, bad, 3, 0], I32)
    t = W.kv_tree(ctx, dev(parents), dev(np.array([0, 6], I32)), dev(np.array([10], I32)), 6)
    raises(W, ctx)
    assert t.masks[:, 0].tolist() == [1, 3, 7, 8, 24, 33] and t.positions.tolist() == [4, 5, 6, 4, 5, 5]


def test_tree_request_with_too_many_nodes(ctx, W):
    parents = np.arange(-1, 69, dtype=I32)
    t = W.kv_tree(ctx, dev(parents), dev(np.array([0, 70], I32)), dev(np.array([100], I32)), 50)
    raises(W, ctx)
    assert t.masks.shape == (70, 1)
    assert t.positions.tolist() == list(range(30, 94)) + [-1] * 6 and not t.masks[64:].any()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
class Case:
    def __init__(self, seed, heads, kvh, d, sep, lens, nodes, page, dtype, q_scale=1.5, spare=2, chain=0.4):
        rng = self.rng = np.random.default_rng(seed)
        self.page, self.dtype, self.lens, self.nodes = page, dtype, list(lens), list(nodes)
        pages = [-(-n // page) for n in lens]
        blocks = sum(pages) + spare

        def rows(shape):
            return rng.standard_normal(shape) * np.where(rng.random(shape[-1]) < 0.03, 5.0, 1.0)

        self.arrays = [x for _ in range(2 if sep else 1) for x in R.quantise(rows((blocks, kvh, page, d)).astype(np.float32))]
        order = rng.permutation(blocks)
        self.table = np.full((len(lens), max(max(pages), 1)), -1, I32)
        for r, p in enumerate(pages):
            self.table[r, :p] = order[sum(pages[:r]):sum(pages[:r + 1])]
        self.cu = starts(nodes)
        self.parents = T.grow(rng, nodes, chain)
        self.masks, self.pos = T.tree(self.parents, self.cu, self.lens, int(self.cu[-1]), -(-max(nodes) // 64))
        self.q = dev(rows((int(self.cu[-1]), heads, d)).astype(np.float32) * np.float32(q_scale)).to(dtype)
        self.sink = rng.standard_normal(heads).astype(np.float32)

    def cache(self, W):
        return W.PagedKvCache(*[dev(x) for x in self.arrays])

    def call(self, W, ctx, cache=None, window=0, first=0, sink=None, **kw):
        return W.kv_tree_attention(ctx, cache or self.cache(W), kw.pop("q", self.q), dev(self.cu), dev(np.array(self.lens, I32)),
                                   dev(self.table), W.KvTree(dev(self.masks), dev(self.pos)), window=window, first=first,
                                   sink=None if sink is None else dev(sink), **kw)

    def check(self, W, ctx, window=0, first=0, sink=False, got=None):
        s = self.sink if sink else None
        got = self.call(W, ctx, window=window, first=first, sink=s) if got is None else got
        ctx.sync()
        k = R.values(*self.arrays[:2])
        v = R.values(*self.arrays[2:]) if len(self.arrays) > 2 else k
        want, smax, vmax = T.attend(self.q.double().cpu().numpy(), k, v, self.cu, self.lens, self.table, self.page,
                                    self.q.shape[2]**-0.5, window, first, s, self.masks, self.pos)
        got = got.double().cpu().numpy()
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        tol = (vmax * 2.0**-22 * (16 + 8 * smax))[..., None] + np.zeros_like(want)
        if self.dtype != F32:
            tol = tol + (vmax * 2.0**-11)[..., None] + UNIT[self.dtype] * np.abs(want) + 2.0**-25
        err = np.where(np.isfinite(want), np.abs(got - want), 0.0)
        tol = np.nan_to_num(tol, nan=np.inf)
        assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())
        return got


LATENT = (64, 1, 512, False)
LAYOUTS = [LATENT, (128, 1, 512, False), (8, 8, 128, True), (28, 4, 128, True), (16, 2, 256, True), (64, 8, 64, True),
           (20, 1, 512, True), (12, 1, 256, False), (34, 2, 64, False), (6, 2, 96, True), (5, 1, 32, False)]


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_attention(ctx, W, layout, dtype):
    # no cached rows, no nodes, trees that end inside a tile and behind it
    Case(1, *layout, [5, 70, 0, 301, 64, 130], [5, 9, 0, 1, 3, 40], 48, dtype).check(W, ctx, sink=layout[0] % 3 != 0)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True), (16, 2, 256, True), (64, 8, 64, True), (6, 2, 96, True)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("nodes", [2, 3])
def test_attention_small_trees(ctx, W, layout, dtype, nodes):
    Case(nodes, *layout, [nodes, 63, 64, 65, 1000], [nodes] * 5, 16, dtype).check(W, ctx)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True), (5, 1, 32, False)], ids=str)
@pytest.mark.parametrize("nodes", [[63], [64], [65, 128], [256, 1]], ids=str)
def test_attention_masks_of_several_words(ctx, W, layout, nodes):
    Case(3, *layout, [n + 37 for n in nodes], nodes, 32, BF16).check(W, ctx)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True), (16, 2, 256, True), (6, 2, 96, True)], ids=str)
@pytest.mark.parametrize("window,first", [(64, 0), (64, 1), (64, 4), (128, 70), (100, 300), (700, 3), (5000, 5)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_attention_window_and_first_tokens(ctx, W, layout, window, first, dtype):
    # chains, so that positions differ within a tree
    Case(window + first, *layout, [9, 127, 128, 129, 640, 1290], [9, 20, 1, 33, 5, 64], 16, dtype, chain=0.9).check(
        W, ctx, window=window, first=first, sink=True)


@pytest.mark.parametrize("layout", [LATENT, (8, 2, 128, True), (6, 2, 96, True)], ids=str)
def test_attention_any_mask(ctx, W, layout):
    # rows that see none of the tree, later nodes, or nothing at all; positions outside the request's rows
    c = Case(4, *layout, [12, 80, 7], [12, 10, 7], 16, F32)
    c.masks = c.rng.integers(-2**63, 2**63 - 1, c.masks.shape)
    c.masks[[0, 13, 22]] = 0
    c.pos = c.rng.integers(-500, 500, c.pos.shape).astype(I32)
    got = c.check(W, ctx, sink=True)
    assert not got[[0, 22]].any()
    c.check(W, ctx, window=64, first=2)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True), (6, 2, 96, True)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_attention_not_finite_rows_reach_only_the_nodes_that_see_them(ctx, W, layout, dtype):
    c = Case(5, *layout, [40, 200], [30, 20], 16, dtype, chain=0.2)
    # node 7's row, and the rows that nobody has
    b, o = c.table[0, 17 // 16], 17 % 16
    c.arrays[-1][b, :, o, 0] = 255
    seen = np.zeros((c.arrays[0].shape[0], 16), bool)
    for r, n in enumerate(c.lens):
        for i in range(n):
            seen[c.table[r, i // 16], i % 16] = True
    for s in c.arrays[1::2]:
        s[np.broadcast_to(~seen[:, None, :, None], s.shape)] = 255
    got = c.check(W, ctx)
    hit = (c.masks[:30, 0] >> 7 & 1).astype(bool)
    assert hit.any() and not hit.all()
    bad = np.isnan(got).any((1, 2))
    np.testing.assert_array_equal(bad[:30], hit)
    assert not bad[30:].any()


def test_attention_of_a_chain_is_causal_attention(ctx, W):
    # A tree that is a line of tokens, on each of the kernels: kv_attention's answer is within
    # the same tolerance of the tree's plain form.  Not bit for bit: a tree's list of rows begins
    # at the first node's window for all of its nodes, so the same rows lie in other tiles and
    # their f32 sums are added in another order.
    for layout, q in ((LATENT, 5), ((28, 4, 128, True), 3), ((6, 2, 96, True), 4)):
        c = Case(6, *layout, [300, 77], [q, q], 16, BF16, chain=1.0)
        c.check(W, ctx, window=64)
        b = W.kv_attention(ctx, c.cache(W), c.q, dev(c.cu), dev(np.array(c.lens, I32)), dev(c.table), window=64)
        c.check(W, ctx, window=64, got=b)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True)], ids=str)
def test_attention_strides_streams_graphs_and_repeats(ctx, W, layout):
    heads, kvh, d, sep = layout
    c = Case(7, *layout, [301, 77, 1500], [20, 1, 9], 16, BF16)
    cache, a = c.cache(W), None
    a = c.call(W, ctx, cache)
    q = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((c.q.shape[0], heads + 3, d + 16), 7.0, dtype=BF16, device="cuda")
    out = wide[:, 1:heads + 1, :d]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c.call(W, ctx, cache, q=q, out=out, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(out, a)
    wide[:, 1:heads + 1, :d] = 7.0
    assert (wide == 7.0).all()
    # out = q, and a captured call
    again = c.q.clone()
    c.call(W, ctx, cache, q=again, out=again)
    assert torch.equal(again, a)
    args = [dev(c.cu), dev(np.array(c.lens, I32)), dev(c.table), W.KvTree(dev(c.masks), dev(c.pos))]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = W.kv_tree_attention(ctx, cache, c.q, *args)
    for _ in range(2):
        got.zero_()
        g.replay()
        assert torch.equal(got, a)
    ctx.sync()
    g.reset()


def test_attention_leaves_tokens_past_the_last_request_alone(ctx, W):
    c = Case(8, *LATENT, [90, 20], [7, 2], 16, F32)
    q = torch.cat([c.q, c.q[:3]])
    out = torch.full_like(q, 5.0)
    tree = W.KvTree(dev(np.concatenate([c.masks, c.masks[:3]])), dev(np.concatenate([c.pos, c.pos[:3]])))
    W.kv_tree_attention(ctx, c.cache(W), q, dev(c.cu), dev(np.array(c.lens, I32)), dev(c.table), tree, out=out)
    ctx.sync()
    assert (out[9:] == 5.0).all()
    c.check(W, ctx, got=out[:9])  # (parts are joined in an order that depends on the number of tokens)


# ---------------------------------------------------------------------------
# accept
# ---------------------------------------------------------------------------
def accept_case(seed, nodes, page, most_len=300, agree=0.6, alphabet=5):
    rng = np.random.default_rng(seed)
    cu, parents = starts(nodes), T.grow(rng, nodes)
    n = int(cu[-1])
    drafts, targets = rng.integers(0, alphabet, n).astype(I32), rng.integers(0, alphabet, n).astype(I32)
    who = np.repeat(cu[:-1], nodes)
    for t in range(n):
        if parents[t] >= 0 and rng.random() < agree:
            targets[who[t] + parents[t]] = drafts[t]
    lens = [k + int(rng.integers(0, most_len)) for k in nodes]
    pages = [-(-x // page) for x in lens]
    table = np.full((len(nodes), max(max(pages), 1) + 1), -1, I32)
    order = rng.permutation(sum(pages) + 5).astype(I32)
    for r, p in enumerate(pages):
        table[r, :p] = order[sum(pages[:r]):sum(pages[:r + 1])]
    free = np.full(sum(pages) + 5, -7, I32)
    free[:5] = order[sum(pages):]
    return parents, drafts, targets, cu, lens, table, free, 5


def run_accept(W, ctx, page, parents, drafts, targets, cu, lens, table, free, top):
    f = dev(free)
    a = W.kv_accept(ctx, page, dev(parents), dev(drafts), dev(targets), dev(cu), dev(np.array(lens, I32)), dev(table), f,
                    dev(np.array([top], I32)))
    return a, f


@pytest.mark.parametrize("nodes", [[1], [0], [7, 0, 3], [16] * 32, [1, 2, 33, 64, 65, 128, 256, 0], [5] * 64, [9] * 65, [3] * 1500],
                         ids=lambda n: f"{len(n)}x{max(n)}")
@pytest.mark.parametrize("page", [1, 16, 48])
def test_accept(ctx, W, nodes, page):
    c = accept_case(len(nodes) + page, nodes, page)
    a, free = run_accept(W, ctx, page, *c)
    ctx.sync()
    counts, path, nxt, lens, stack, top = T.accept(page, *c)
    assert a.counts.tolist() == counts and a.next_tokens.tolist() == nxt and a.kv_lens.tolist() == lens
    np.testing.assert_array_equal(a.path.cpu().numpy(), path)
    np.testing.assert_array_equal(free.cpu().numpy(), stack)
    assert a.free_top.tolist() == [top]


def test_accept_takes_the_child_of_least_index(ctx, W):
    # two equal drafts below node 0; the second has the longer agreement
    parents = np.array([-1, 0, 0, 2], I32)
    c = (parents, np.array([1, 9, 9, 4], I32), np.array([9, 8, 4, 6], I32), np.array([0, 4], I32), [20], np.array([[3, 1]], I32),
         np.full(4, -1, I32), 0)
    a, free = run_accept(W, ctx, 16, *c)
    ctx.sync()
    assert (a.counts.tolist(), a.path.tolist(), a.next_tokens.tolist()) == ([2], [0, 1, -1, -1], [8])
    # 18 rows still need both pages
    assert a.kv_lens.tolist() == [18] and a.free_top.tolist() == [0]


def test_accept_other_roots_and_bad_parents_are_on_no_path(ctx, W):
    parents = np.array([-1, -1, 5, 0], I32)
    c = (parents, np.array([1, 2, 2, 2], I32), np.array([2, 2, 2, 7], I32), np.array([0, 4], I32), [4], np.array([[0]], I32),
         np.zeros(1, I32), 0)
    a, _ = run_accept(W, ctx, 16, *c)
    raises(W, ctx)
    assert (a.counts.tolist(), a.path.tolist(), a.next_tokens.tolist()) == ([2], [0, 3, -1, -1], [7])


@pytest.mark.parametrize("requests", [3, 70])
@pytest.mark.parametrize("bad", ["capacity", "top", "negative top"])
def test_accept_that_does_not_fit_the_stack_changes_nothing(ctx, W, requests, bad):
    c = list(accept_case(5, [20] * requests, 4, agree=0.0))
    if bad == "capacity":
        c[6] = c[6][:7]
    else:
        c[7] = len(c[6]) + 1 if bad == "top" else -1
    a, free = run_accept(W, ctx, 4, *c)
    raises(W, ctx)
    assert not a.counts.any() and (a.path == -1).all() and (a.next_tokens == -1).all()
    assert a.kv_lens.tolist() == c[4] and a.free_top.tolist() == [c[7]]
    np.testing.assert_array_equal(free.cpu().numpy(), c[6])


def test_accept_a_request_that_does_not_fit_is_left_alone(ctx, W):
    parents, drafts, targets, cu, lens, table, free, top = accept_case(6, [4, 6, 300, 5], 8)
    lens = list(lens)
    lens[0], lens[3] = 3, 8 * table.shape[1] + 1  # fewer rows than nodes; more than the table holds
    a, f = run_accept(W, ctx, 8, parents, drafts, targets, cu, lens, table, free, top)
    raises(W, ctx)
    t0, t1 = cu[1], cu[2]
    one = T.accept(8, parents[t0:t1], drafts[t0:t1], targets[t0:t1], [0, 6], [lens[1]], table[1:2], free, top)
    assert a.counts.tolist() == [0, one[0][0], 0, 0] and a.next_tokens.tolist() == [-1, one[2][0], -1, -1]
    assert a.kv_lens.tolist() == [lens[0], one[3][0], lens[2], lens[3]] and a.free_top.tolist() == [one[5]]
    np.testing.assert_array_equal(a.path.cpu().numpy()[t0:t1], one[1])
    assert (a.path[:4] == -1).all() and (a.path[10:] == -1).all()
    np.testing.assert_array_equal(f.cpu().numpy(), one[4])


def test_accept_tokens_of_no_request(ctx, W):
    parents, drafts, targets, cu, lens, table, free, top = accept_case(7, [4, 6], 8)
    pad = np.zeros(1100, I32)
    a, _ = run_accept(W, ctx, 8, *(np.concatenate([x, pad]) for x in (parents, drafts, targets)), cu, lens, table, free, top)
    ctx.sync()
    assert a.path[:10].tolist() == T.accept(8, parents, drafts, targets, cu, lens, table, free, top)[1].tolist()
    assert (a.path[10:] == -1).all()


# ---------------------------------------------------------------------------
# commit
# ---------------------------------------------------------------------------
def commit_case(seed, kvh, d, sep, nodes, page, layers=1, share=1.0):
    c = Case(seed, kvh, kvh, d, sep, [n + 5 + 31 * i for i, n in enumerate(nodes)], nodes, page, F32)
    path, counts = np.full(int(c.cu[-1]), -1, I32), []
    for r, n in enumerate(nodes):
        k = 0 if n == 0 else 1 + int(c.rng.integers(0, max(1, int(share * n))))
        path[c.cu[r]:c.cu[r] + k] = np.concatenate([[0], 1 + np.sort(c.rng.permutation(n - 1)[:k - 1])]) if k else []
        counts.append(k)
    return c, counts, path


@pytest.mark.parametrize("kvh,d,sep", [(1, 512, False), (4, 128, True), (2, 256, False), (3, 96, True), (8, 64, True), (1, 32, True),
                                       (43, 512, False)])
@pytest.mark.parametrize("nodes", [[1], [9, 0, 2, 33], [256, 100]], ids=str)
@pytest.mark.parametrize("page", [1, 16, 24])
def test_commit(ctx, W, kvh, d, sep, nodes, page):
    if kvh == 43 and page == 1:
        page = 8
    c, counts, path = commit_case(kvh + page, kvh, d, sep, nodes, page)
    cache = c.cache(W)
    W.kv_commit(ctx, cache, dev(np.array(counts, I32)), dev(path), dev(c.cu), dev(np.array(c.lens, I32)), dev(c.table))
    ctx.sync()
    want = T.commit(c.arrays, counts, path, c.cu, c.lens, c.table, page)
    for x, y in zip((cache.keys, cache.key_scales, cache.values, cache.value_scales), want):
        np.testing.assert_array_equal(x.cpu().numpy(), y)


def test_commit_layers_inside_a_block_and_apart(ctx, W):
    # a pool [blocks, layers, 1, page, ..]: all layers at once, or one after the other
    c, counts, path = commit_case(9, 3, 128, False, [12, 5], 16)
    args = [dev(x) for x in (np.array(counts, I32), path, c.cu, np.array(c.lens, I32), c.table)]
    whole = c.cache(W)
    W.kv_commit(ctx, whole, *args)
    codes, scales = (dev(x) for x in c.arrays)
    for i in range(3):
        W.kv_commit(ctx, W.PagedKvCache(codes[:, i:i + 1], scales[:, i:i + 1]), *args)
    ctx.sync()
    assert torch.equal(codes, whole.keys) and torch.equal(scales, whole.key_scales)


@pytest.mark.parametrize("bad", ["repeat", "falls", "early", "past", "count", "negative count", "length", "long"])
def test_commit_paths_and_lengths_that_do_not_fit(ctx, W, bad):
    c, counts, path = commit_case(10, 2, 128, True, [10, 10], 16)
    counts, lens = [4, 4], list(c.lens)
    path[:] = -1
    path[:4], path[10:14] = [0, 2, 5, 9], [0, 3, 4, 8]
    if bad == "repeat":
        path[2] = 2
    elif bad == "falls":
        path[3] = 3
    elif bad == "early":
        path[1] = 0
    elif bad == "past":
        path[3] = 10
    elif bad == "count":
        counts[0] = 11
    elif bad == "negative count":
        counts[0] = -1
    elif bad == "length":
        lens[0] = 9
    else:
        lens[0] = 16 * c.table.shape[1] + 1
    cache = c.cache(W)
    W.kv_commit(ctx, cache, dev(np.array(counts, I32)), dev(path), dev(c.cu), dev(np.array(lens, I32)), dev(c.table))
    raises(W, ctx)
    want = T.commit(c.arrays, [0, 4], path, c.cu, c.lens, c.table, 16)  # the other request's rows still move
    np.testing.assert_array_equal(cache.keys.cpu().numpy(), want[0])
    np.testing.assert_array_equal(cache.value_scales.cpu().numpy(), want[3])


def test_commit_a_block_outside_the_pool(ctx, W):
    c, counts, path = commit_case(11, 1, 512, False, [40], 16)
    counts, path[:] = [3], -1
    path[:3] = [0, 20, 39]
    c.table[0, (c.lens[0] - 40 + 20) // 16] = 10**6
    cache = c.cache(W)
    W.kv_commit(ctx, cache, dev(np.array(counts, I32)), dev(path), dev(c.cu), dev(np.array(c.lens, I32)), dev(c.table))
    raises(W, ctx)
    base = c.lens[0] - 40
    want = c.arrays[0].copy()
    want[c.table[0, (base + 2) // 16], :, (base + 2) % 16] = c.arrays[0][c.table[0, (base + 39) // 16], :, (base + 39) % 16]
    np.testing.assert_array_equal(cache.keys.cpu().numpy(), want)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def refused(W, kind, fn, *a, **kw):
    with pytest.raises(W.WohperError) as e:
        fn(*a, **kw)
    assert e.value.kind == kind, e.value


def test_refusals(ctx, W):
    c = Case(12, 8, 2, 128, True, [40, 30], [6, 5], 16, BF16)
    cache, cu, lens, table = c.cache(W), dev(c.cu), dev(np.array(c.lens, I32)), dev(c.table)
    tree = W.KvTree(dev(c.masks), dev(c.pos))
    parents = dev(c.parents)
    at = W.kv_tree_attention
    refused(W, "InvalidShape", at, ctx, cache, c.q, cu, lens, table, W.KvTree(tree.masks[:-1], tree.positions))
    refused(W, "InvalidShape", at, ctx, cache, c.q, cu, lens, table, W.KvTree(tree.masks, tree.positions[:-1]))
    refused(W, "InvalidShape", at, ctx, cache, c.q, cu, lens, table, W.KvTree(tree.masks.repeat(1, 5), tree.positions))
    refused(W, "Unsupported", at, ctx, cache, c.q, cu, lens, table, W.KvTree(tree.masks.int(), tree.positions))
    refused(W, "InvalidPointer", at, ctx, cache, c.q, cu, lens, table, W.KvTree(tree.masks.cpu(), tree.positions))
    refused(W, "Unsupported", at, ctx, cache, c.q, cu, lens, table, tree, window=63)
    refused(W, "Unsupported", at, ctx, cache, c.q, cu, lens, table, W.KvTree(tree.masks.repeat(1, 2), tree.positions), window=127)
    for most in (0, 257):
        refused(W, "Unsupported", W.kv_tree, ctx, parents, cu, lens, most)
    refused(W, "InvalidShape", W.kv_tree, ctx, parents, cu[:-1], lens, 6)
    refused(W, "Unsupported", W.kv_tree, ctx, parents.long(), cu, lens, 6)
    free, top = torch.zeros(9, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    ok = [parents, parents, parents, cu, lens, table, free, top]
    for i, x in ((1, parents[:-1]), (2, parents[:-1]), (3, cu[1:]), (5, table[:1]), (7, free)):
        refused(W, "InvalidShape", W.kv_accept, ctx, 16, *ok[:i], x, *ok[i + 1:])
    refused(W, "EmptyShape", W.kv_accept, ctx, 0, *ok)
    refused(W, "Unsupported", W.kv_accept, ctx, 16, *ok[:1], parents.long(), *ok[2:])
    refused(W, "InvalidShape", W.kv_commit, ctx, cache, lens[:1], parents, cu, lens, table)
    refused(W, "InvalidPointer", W.kv_commit, ctx, cache, lens.cpu(), parents, cu, lens, table)
    ctx.sync()


def test_no_tokens(ctx, W):
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    cu, lens = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([5, 0], dtype=torch.int32, device="cuda")
    table, free = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    t = W.kv_tree(ctx, none, cu, lens, 16)
    assert t.masks.shape == (0, 1) and t.positions.shape == (0,)
    cache = W.PagedKvCache.empty(4, 16, 1, 512)
    out = W.kv_tree_attention(ctx, cache, torch.zeros(0, 64, 512, device="cuda"), cu, lens, table, t)
    assert out.shape == (0, 64, 512)
    a = W.kv_accept(ctx, 16, none, none, none, cu, lens, table, free, free[:1])
    W.kv_commit(ctx, cache, a.counts, a.path, cu, lens, table)
    ctx.sync()
    assert a.counts.tolist() == [0, 0] and a.kv_lens.tolist() == [5, 0] and a.free_top.tolist() == [0]
