"""The paged cache's attention where a CTA of the tensor-core kernel takes many short
items one after the other, and where items end early, begin in bad blocks or are
computed again.  Cases, plain 64-bit form and tolerances are those of
tests/test_gpu_kvcache.py."""
from __future__ import annotations

import numpy as np
import pytest

from tests import kv_reference as R
from tests.test_gpu_kvcache import BF16, F32, Case, ctx, dev, tolerance, W  # noqa: F401 (fixtures)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# enough rows to a kv head for the tensor-core kernel: above 24 / 48 (64 wide) and
# 20 / 40 (128 wide) of f32 / bf16
@pytest.mark.parametrize("heads,d,dtype", [(29, 64, F32), (64, 64, F32), (57, 64, BF16), (27, 128, F32),
                                           (64, 128, F32), (48, 128, BF16), (64, 128, BF16)], ids=str)
@pytest.mark.parametrize("sep", [False, True], ids=["latent", "values"])
def test_every_item_is_scored_with_its_own_queries(ctx, W, heads, d, dtype, sep):  # noqa: F811
    # 600 items of one or two tiles, several to a CTA: each needs its own queries in
    # shared memory, all of their rows, before its first product
    rng = np.random.default_rng(heads + d)
    lens = rng.integers(1, 100, 600).tolist()
    c = Case(31, heads, 1, d, sep, lens, [1] * 600, 16, dtype)
    got, _ = c.check(W, ctx)
    args = (c.cache(W), c.q, dev(c.cu), dev(np.array(lens, np.int32)), dev(c.table))
    for _ in range(5):
        again = W.kv_attention(ctx, *args)
        np.testing.assert_array_equal(again.double().cpu().numpy(), got)
    ctx.sync()


@pytest.mark.parametrize("layout", [(64, 1, 512, False), (28, 4, 128, True), (64, 1, 128, True), (16, 2, 256, True),
                                    (6, 2, 96, True)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_out_may_be_q(ctx, W, layout, dtype):  # noqa: F811
    # many items that lie in one CTA, some computed again: a query that is not finite, a
    # scale byte that f16 does not hold; and one long request that is split
    lens = [40] * 300 + [3000]

    def spoil(c):
        c.q[::7, 0, 3] = float("nan")
        for r in range(0, 300, 5):
            for s in c.scales:
                s[c.table[r, 1], :, 2, 0] = 90

    c = Case(32, *layout, lens, [1] * 301, 16, dtype, spoil=spoil)
    args = (dev(c.cu), dev(np.array(lens, np.int32)), dev(c.table))
    cache = c.cache(W)
    want = W.kv_attention(ctx, cache, c.q, *args)
    q = c.q.clone()
    got = W.kv_attention(ctx, cache, q, *args, out=q)
    ctx.sync()
    assert got is q
    np.testing.assert_array_equal(got.double().cpu().numpy(), want.double().cpu().numpy())
    assert torch.isfinite(want[:, 1:]).all() and not torch.isfinite(want[::7, 0]).any()


@pytest.mark.parametrize("layout", [(64, 1, 512, False), (28, 4, 128, True), (64, 1, 128, True), (64, 1, 64, False),
                                    (16, 2, 256, True), (6, 2, 96, True)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("sink", [False, True], ids=["", "sink"])
def test_rows_of_bad_blocks_count_as_not_seen(ctx, W, layout, dtype, sink):  # noqa: F811
    # runs of bad pages (16 rows) at the front, in the middle, at the end and everywhere,
    # so that a CTA's first tiles hold no row, over items of one CTA and of several
    lens, page = [200, 100, 64] + [3000] * 14 + [70], 16
    c = Case(33, *layout, lens, [1] * len(lens), page, dtype)
    bad = [[0, 1, 2, 3, 4], [6], [0, 1, 2, 3]]
    bad += [sorted(c.rng.choice(187, 90, False)) if r % 3 else list(range(r, r + 100)) for r in range(14)]
    bad += [[0, 2, 3]]
    lens_d = dev(np.array(lens, np.int32))
    table = c.table.copy()
    for r, b in enumerate(bad):
        table[r, b] = -1 if r % 2 else c.codes[0].shape[0] + r
    got = W.kv_attention(ctx, c.cache(W), c.q, dev(c.cu), lens_d, dev(table),
                         sink=dev(c.sink) if sink else None)
    with pytest.raises(W.WohperError, match="DeviceArg"):
        ctx.sync()
    # the plain form over the pages that are there: one query, which sees all of them
    for r, b in enumerate(bad):
        left = np.delete(c.table[r], b)
        c.table[r], c.table[r, :len(left)] = -1, left
        c.lens[r] = lens[r] - sum(min(page, lens[r] - page * i) for i in b)
    want, smax, vmax = c.want(layout[2] ** -0.5, sink=c.sink if sink else None)
    ratio = np.abs(got.double().cpu().numpy() - want) / np.maximum(tolerance(want, smax, vmax, dtype), 1e-300)
    assert (ratio <= 1).all(), np.argwhere(ratio.max((1, 2)) > 1).ravel()


@pytest.mark.parametrize("page", [1, 7, 16, 24, 100])
@pytest.mark.parametrize("layout", [(8, 2, 128, True), (28, 4, 128, True), (8, 2, 64, False), (4, 2, 256, True),
                                    (64, 1, 512, False), (64, 1, 128, True), (6, 2, 96, True)], ids=str)
@pytest.mark.parametrize("window,first", [(40, 0), (40, 5), (130, 33)])
def test_pages_that_no_query_sees_need_no_block(ctx, W, page, layout, window, first):  # noqa: F811
    # a server gives back the pages behind the window: their entries are -1 (or stale
    # ids past a pool that shrank), and the step is still an ordinary one
    lens, qs = [640, 129, 333, 41, 1, 1000], [1, 3, 1, 1, 1, 2]
    c = Case(34 + page, *layout, lens, qs, page, BF16)
    table = c.table.copy()
    for r, (n, q) in enumerate(zip(lens, qs)):
        seen = [i for i in range(n) if i > n - q - window or i < first]
        keep = {i // page for i in seen}
        for p in range(table.shape[1]):
            if p not in keep:
                table[r, p] = -1 if (r + p) % 2 else 1 << 30
    c.table, full = table, c.table
    lens_d = dev(np.array(lens, np.int32))
    got = W.kv_attention(ctx, c.cache(W), c.q, dev(c.cu), lens_d, dev(c.table), window=window, first=first)
    ctx.sync()  # nothing recorded
    want, smax, vmax = c.want(layout[2] ** -0.5, window, first)
    assert (np.abs(got.double().cpu().numpy() - want) <= tolerance(want, smax, vmax, BF16)).all()
    again = W.kv_attention(ctx, c.cache(W), c.q, dev(c.cu), lens_d, dev(full), window=window, first=first)
    assert torch.equal(got, again)


def test_a_context_of_another_gpu_is_refused(ctx, W):  # noqa: F811
    class Other:
        device, handle = ctx.device + 1, ctx.handle

    cache = W.PagedKvCache.empty(4, 16, 1, 64)
    slots, lens = torch.arange(2, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    table, q = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, 64, device="cuda")
    for call in (lambda: W.kv_append(Other, cache, slots, q[:, :1].contiguous()), lambda: W.kv_gather(Other, cache, slots),
                 lambda: W.kv_attention(Other, cache, q, None, lens, table),
                 lambda: W.kv_plan(Other, 16, lens, lens, table, slots.int(), lens[:1], 2)):
        with pytest.raises(W.WohperError) as e:
            call()
        assert e.value.kind == "InvalidPointer"
    ctx.sync()


def test_a_scratch_that_is_not_dense_memory_of_the_gpu_is_refused(ctx, W):  # noqa: F811
    cache = W.PagedKvCache.empty(4, 16, 2, 128, True)
    lens, table = torch.ones(2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 4, 128, device="cuda")
    n = 1 << 24  # more than the call needs
    for kind, scratch in (("InvalidPointer", torch.empty(n, dtype=torch.uint8)),
                          ("InvalidShape", torch.empty(1, dtype=torch.uint8, device="cuda").expand(n)),
                          ("InvalidShape", torch.empty(2 * n, dtype=torch.uint8, device="cuda")[::2])):
        with pytest.raises(W.WohperError) as e:
            W.kv_attention(ctx, cache, q, None, lens, table, scratch=scratch)
        assert e.value.kind == kind
    ok = torch.empty(n // 4, 4, dtype=torch.uint8, device="cuda")
    assert W.kv_attention(ctx, cache, q, None, lens, table, scratch=ok).shape == q.shape
    ctx.sync()


@pytest.mark.parametrize("layout", [(26, 1, 64, False), (22, 1, 128, True), (3, 1, 512, False)], ids=str)
@pytest.mark.parametrize("sink", [False, True], ids=["", "sink"])
def test_items_of_more_tiles_than_a_sum_runs_through(ctx, W, layout, sink):  # noqa: F811
    # 160 items of up to 47 tiles and two long ones: some in one CTA, some in several, sums
    # put aside after 32 tiles; rows to be computed again because of the first, the last or a
    # middle tile; a largest score that comes early, late, or not at all
    lens = ([3000, 2049, 2048, 2900] * 40) + [9000, 12000]

    def spoil(c):
        for r, p in ((3, 0), (8, 100), (13, 180), (160, 0), (161, 700)):
            c.scales[0][c.table[r, p], :, 2, 0] = 90
        c.q[20, 1, 3] = float("inf")
        for r, i in ((30, 5), (31, 2040), (32, 2999), (161, 11000)):
            row = c.q[r, 0].float().cpu().numpy()
            cc, ss = R.quantise(row * 2)
            c.codes[0][c.table[r, i // 16], :, i % 16], c.scales[0][c.table[r, i // 16], :, i % 16] = cc, ss

    c = Case(35, *layout, lens, [1] * len(lens), 16, F32, spoil=spoil)
    args = (c.cache(W), c.q, dev(c.cu), dev(np.array(lens, np.int32)), dev(c.table))
    kw = dict(sink=dev(c.sink) if sink else None)
    got = W.kv_attention(ctx, *args, **kw)
    for _ in range(3):
        assert torch.equal(got.nan_to_num(), W.kv_attention(ctx, *args, **kw).nan_to_num())
    q = c.q.clone()
    W.kv_attention(ctx, args[0], q, *args[2:], **kw, out=q)
    ctx.sync()
    assert torch.equal(got.nan_to_num(), q.nan_to_num()) and torch.isnan(got[20, 1]).all()
    c.q[20, 1] = 1.0  # its own row is not compared
    want, smax, vmax = c.want(layout[2] ** -0.5, sink=c.sink if sink else None)
    ratio = np.abs(got.double().cpu().numpy() - want) / np.maximum(tolerance(want, smax, vmax, F32), 1e-300)
    ratio[20, 1] = 0
    assert (ratio <= 1).all(), np.argwhere(~(ratio.max((1, 2)) <= 1)).ravel()


def test_numbers_past_32_bits_are_refused(ctx, W):  # noqa: F811
    # the C calls take int: 2^32 + n would arrive as n
    cache = W.PagedKvCache.empty(4, 16, 1, 64)
    lens, table = torch.ones(2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 3, 64, device="cuda")
    free = torch.arange(4, dtype=torch.int32, device="cuda")
    for n in (1 << 31, 1 << 32, (1 << 32) + 16, 1 << 63):
        for call in (lambda: W.kv_attention(ctx, cache, q, None, lens, table, window=n),
                     lambda: W.kv_attention(ctx, cache, q, None, lens, table, first=n),
                     lambda: W.kv_plan(ctx, n, lens, lens, table, free, lens[:1], 2),
                     lambda: W.kv_plan(ctx, 16, lens, lens, table, free, lens[:1], n)):
            with pytest.raises(W.WohperError) as e:
                call()
            assert e.value.kind == "InvalidShape"
    most = (1 << 31) - 1
    a = W.kv_attention(ctx, cache, q, None, lens, table, window=most, first=most)
    assert torch.equal(a, W.kv_attention(ctx, cache, q, None, lens, table))
    ctx.sync()


def test_an_out_whose_rows_share_memory_is_refused(ctx, W):  # noqa: F811
    cache = W.PagedKvCache.empty(4, 16, 1, 64)
    lens, table = torch.ones(2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 3, 64, device="cuda")
    for out in (torch.empty(1, 3, 64, device="cuda").expand(2, 3, 64), torch.empty(2, 1, 64, device="cuda").expand(2, 3, 64)):
        with pytest.raises(W.WohperError) as e:
            W.kv_attention(ctx, cache, q, None, lens, table, out=out)
        assert e.value.kind == "InvalidShape"
    # where there is one token, one head, a stride means nothing; queries may share memory
    one = torch.empty(1, 1, 64, device="cuda").expand(1, 1, 64)
    W.kv_attention(ctx, cache, q[:1, :1].contiguous(), None, lens[:1], table[:1], out=one)
    W.kv_attention(ctx, cache, q[:1].expand(2, 3, 64), None, lens, table)
    ctx.sync()
