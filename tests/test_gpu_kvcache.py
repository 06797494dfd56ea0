"""The paged 4-bit key/value cache on the GPU: plan, append, gather and attention
against plain 64-bit forms (tests/kv_reference.py), and what they refuse.

Tolerances of the attention, per output element, with V the largest |value| and S
the largest |score| that the query row sees:
 - f32: V * 2^-22 * (16 + 8 S).  A score is a sum of up to 512 products of which
   each partial sum rounds by 2^-24 of its size: a few 2^-22 of S in practice,
   which moves each weight by that share; exp2's argument rounds by 2^-24 of
   1.44 S, exp2 itself by 2^-22, and the weights' sums by a few 2^-24.
 - bf16, f16: as f32, plus V * 2^-11 for weights held in 11 bits (the error of a
   weight is at most 2^-11 of it, so that of the mean at most 2^-11 V), plus the
   output's own rounding, the type's unit roundoff (8 and 11 significant bits:
   2^-8 and 2^-11 of it; f16 adds 2^-25 for subnormal outputs).
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import kv_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 0.0, BF16: 2.0**-8, F16: 2.0**-11}


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


def make_rows(rng, shape):
    gain = np.where(rng.random(shape[-1]) < 0.03, 5.0, 1.0)
    return (rng.standard_normal(shape) * gain).astype(np.float32)


def tolerance(want, smax, vmax, dtype):
    t = (vmax * 2.0**-22 * (16 + 8 * smax))[..., None] + np.zeros_like(want)
    if dtype != F32:
        t = t + (vmax * 2.0**-11)[..., None] + UNIT[dtype] * np.abs(want) + 2.0**-25
    return t


class Case:
    """A pool with shuffled blocks, requests of given lengths and their queries."""

    def __init__(self, seed, heads, kvh, d, sep, lens, qs, page, dtype, q_scale=1.5, spare=2,
                 spoil=None):
        rng = np.random.default_rng(seed)
        self.rng, self.page, self.dtype = rng, page, dtype
        pages = [max(0, -(-n // page)) for n in lens]
        blocks = sum(pages) + spare
        self.codes, self.scales = [], []
        for _ in range(2 if sep else 1):
            c, s = R.quantise(make_rows(rng, (blocks, kvh, page, d)))
            self.codes.append(c)
            self.scales.append(s)
        order = rng.permutation(blocks)
        self.table = np.full((len(lens), max(max(pages), 1)), -1, np.int32)
        used = 0
        for r, p in enumerate(pages):
            self.table[r, :p] = order[used:used + p]
            used += p
        self.lens = list(lens)
        self.cu = np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)
        self.q = dev(make_rows(rng, (int(self.cu[-1]), heads, d)) * np.float32(q_scale)).to(dtype)
        self.sink = rng.standard_normal(heads).astype(np.float32)
        if spoil:
            spoil(self)

    def cache(self, W):
        t = [dev(x) for pair in zip(self.codes, self.scales) for x in pair]
        return W.PagedKvCache(*t)

    def want(self, scale, window=0, first=0, sink=None):
        k = R.values(self.codes[0], self.scales[0])
        v = k if len(self.codes) == 1 else R.values(self.codes[1], self.scales[1])
        return R.attend(self.q.double().cpu().numpy(), k, v, self.cu, self.lens, self.table,
                        self.page, scale, window, first, sink)

    def check(self, W, ctx, window=0, first=0, sink=False, scale=None, **kw):
        d = self.q.shape[2]
        scale = d**-0.5 if scale is None else scale
        s = self.sink if sink else None
        got = W.kv_attention(ctx, self.cache(W), self.q, dev(self.cu),
                             dev(np.array(self.lens, np.int32)), dev(self.table), scale=scale,
                             window=window, first=first, sink=None if s is None else dev(s), **kw)
        ctx.sync()
        want, smax, vmax = self.want(scale, window, first, s)
        got = got.double().cpu().numpy()
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        fine = np.isfinite(want)
        err = np.where(fine, np.abs(got - want), 0.0)
        tol = np.nan_to_num(tolerance(want, smax, vmax, self.dtype), nan=np.inf)
        assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())
        return got, want


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
LATENT = (64, 1, 512, False)
LAYOUTS = [LATENT, (128, 1, 512, False), (8, 8, 128, True), (28, 4, 128, True), (16, 2, 256, True),
           (64, 8, 64, True), (20, 1, 512, True), (12, 1, 256, False), (80, 2, 128, True),
           (34, 2, 64, False), (6, 2, 96, True), (5, 1, 32, False)]
LENGTHS = [[1], [0, 1, 2, 63, 64, 65, 0], [127, 128, 129, 191], [1000, 3, 517], [2500]]


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_attention_one_token_each(ctx, W, layout, lens, dtype):
    c = Case(sum(lens) + layout[0], *layout, lens, [1] * len(lens), 16, dtype)
    c.check(W, ctx, sink=layout[0] % 3 != 0)


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("dtype", [F32, F16], ids=str)
def test_attention_several_tokens_each(ctx, W, layout, dtype):
    # causal inside the step; more queries than rows, no queries, no rows
    lens, qs = [5, 66, 300, 2, 0, 130, 64], [5, 3, 0, 4, 2, 8, 1]
    c = Case(7, *layout, lens, qs, 48, dtype)
    c.check(W, ctx, sink=True)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True), (64, 8, 64, True)], ids=str)
def test_attention_prompt_of_many_tokens(ctx, W, layout):
    heads, kvh, d, sep = layout
    c = Case(8, *layout, [150, 201], [150, 37], 64, BF16)
    c.check(W, ctx)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True), (16, 2, 256, True)], ids=str)
@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (64, 4), (128, 4), (128, 70), (100, 300),
                                          (700, 3), (5000, 5)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_attention_window_and_first_tokens(ctx, W, layout, window, first, dtype):
    lens, qs = [1, 127, 128, 129, 640, 1290, 200], [1, 1, 1, 1, 5, 1, 70]
    c = Case(window + first, *layout, lens, qs, 16, dtype)
    c.check(W, ctx, window=window, first=first, sink=True)


@pytest.mark.parametrize("page", [1, 7, 16, 48, 64, 100, 256])
@pytest.mark.parametrize("layout", [LATENT, (8, 2, 128, True)], ids=str)
def test_attention_page_sizes(ctx, W, layout, page):
    c = Case(page, *layout, [333, page, page + 1, max(1, page - 1)], [1, 1, 1, 1], page, F32)
    c.check(W, ctx)


@pytest.mark.parametrize("layout", [LATENT, (8, 2, 128, True)], ids=str)
def test_attention_many_requests(ctx, W, layout):
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 300, 700).tolist()
    c = Case(9, *layout, lens, [1] * 700, 32, BF16)
    c.check(W, ctx)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_attention_more_requests_than_a_cta_has_threads(ctx, W, dtype):
    rng = np.random.default_rng(4)
    lens, qs = rng.integers(0, 90, 1900).tolist(), rng.integers(0, 2, 1900).tolist()
    lens[1500] = 700
    c = Case(24, 9, 1, 512, False, lens, qs, 32, dtype)
    c.check(W, ctx, window=200, first=2)


@pytest.mark.parametrize("layout", [LATENT, (8, 2, 128, True), (32, 8, 128, True)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_attention_long_context(ctx, W, layout, dtype):
    c = Case(10, *layout, [20011], [1], 64, dtype)
    c.check(W, ctx, sink=True)


@pytest.mark.parametrize("layout", [LATENT, (8, 2, 128, True), (6, 2, 96, True)], ids=str)
@pytest.mark.parametrize("q_scale", [0.0, 1e-30, 40.0, 1e6])
def test_attention_peaked_and_flat_scores(ctx, W, layout, q_scale):
    c = Case(11, *layout, [700, 90], [1, 2], 16, F32, q_scale=q_scale)
    c.check(W, ctx, sink=q_scale < 1e5)


@pytest.mark.parametrize("layout", [LATENT, (8, 2, 128, True)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_attention_rising_scores_rescale_the_running_sums(ctx, W, layout, dtype):
    # the running maximum grows by about 3 at each row block
    def spoil(c):
        d = c.q.shape[2]
        u = np.sign(c.rng.standard_normal(d)).astype(np.float32)
        n = c.lens[0]
        for i in range(n):
            row = (u * (i // 32) * 0.04 + c.rng.standard_normal(d) * 0.05).astype(np.float32)
            cc, ss = R.quantise(row)
            b, o = c.table[0, i // c.page], i % c.page
            c.codes[0][b, :, o], c.scales[0][b, :, o] = cc, ss
        c.q = torch.from_numpy(np.broadcast_to(u * 4, tuple(c.q.shape)).copy()).cuda().to(c.dtype)

    c = Case(12, *layout, [1500], [1], 16, dtype, spoil=spoil)
    c.check(W, ctx)


def poison_unseen(c, keep):
    """Not-finite scale bytes in every row that `keep(r, i)` says nobody sees."""
    seen = np.zeros((c.codes[0].shape[0], c.page), bool)
    for r, n in enumerate(c.lens):
        for i in range(n):
            if keep(r, i):
                seen[c.table[r, i // c.page], i % c.page] = True
    for s in c.scales:
        s[np.broadcast_to(~seen[:, None, :, None], s.shape)] = 255


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("window,first", [(0, 0), (64, 4)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_attention_not_finite_rows_in_unseen_places(ctx, W, layout, window, first, dtype):
    lens = [77, 200, 0, 1, 129]

    def spoil(c):
        poison_unseen(c, lambda r, i: not window or i > lens[r] - 1 - window or i < first)

    c = Case(13, *layout, lens, [1] * 5, 16, dtype, spoil=spoil)
    got, _ = c.check(W, ctx, window=window, first=first)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True), (6, 2, 96, True)], ids=str)
@pytest.mark.parametrize("window", [0, 20])
def test_attention_not_finite_row_reaches_only_the_queries_that_see_it(ctx, W, layout, window):
    def spoil(c):
        # row 95 of request 0: seen by the queries at 95.. (and, in a window, only to 114)
        b, o = c.table[0, 95 // 16], 95 % 16
        c.scales[-1][b, 0, o, 0] = 255

    c = Case(14, *layout, [120, 40], [30, 1], 16, F32, spoil=spoil)
    got, want = c.check(W, ctx, window=window)
    assert np.isnan(want).any() and np.isfinite(want[:5]).all() and np.isfinite(want[30]).all()


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True), (16, 2, 256, True)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("lo,hi", [(60, 120), (1, 40), (120, 160), (100, 145), (0, 1)])
def test_attention_scale_bytes_over_the_whole_range(ctx, W, layout, dtype, lo, hi):
    def spoil(c):
        for s in c.scales:
            s[...] = c.rng.integers(lo, hi, s.shape)
        c.q = c.q * 2.0 ** (127 - max(hi, 40))  # keeps the scores in a softmax's range

    c = Case(15, *layout, [150, 31], [1, 2], 16, dtype, spoil=spoil)
    c.check(W, ctx)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True)], ids=str)
def test_attention_one_block_out_of_range_among_ordinary_ones(ctx, W, layout):
    def spoil(c):
        for s in c.scales:
            s[c.table[0, 3], 0, 5, 1] = 150
            s[c.table[1, 0], -1, 2, 0] = 90

    c = Case(16, *layout, [150, 31, 400], [1, 2, 1], 16, F32, q_scale=1e-4, spoil=spoil)
    c.check(W, ctx)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True)], ids=str)
def test_attention_query_rows_that_are_not_finite_or_tiny(ctx, W, layout):
    def spoil(c):
        c.q[0, 1, 3] = float("nan")
        c.q[1, 0, 0] = float("inf")
        c.q[2, 2] = 0.0
        c.q[2, 3] *= 1e-38
        c.q[0, 0, :4] *= 1e-6

    c = Case(17, *layout, [90, 70], [2, 1], 16, F32, spoil=spoil)
    k = R.values(c.codes[0], c.scales[0])
    got = W.kv_attention(ctx, c.cache(W), c.q, dev(c.cu), dev(np.array(c.lens, np.int32)),
                         dev(c.table)).double().cpu().numpy()
    ctx.sync()
    assert k.size and np.isnan(got[0, 1]).all() and np.isnan(got[1, 0]).all()
    c.q[0, 1] = 1.0
    c.q[1, 0] = 1.0
    want, smax, vmax = c.want(c.q.shape[2] ** -0.5)
    tol = tolerance(want, smax, vmax, F32)
    skip = np.zeros(want.shape[:2], bool)
    skip[0, 1] = skip[1, 0] = True
    assert (np.abs(got - want)[~skip] <= tol[~skip]).all()


@pytest.mark.parametrize("sink", ["lowest", "-inf", "high"])
@pytest.mark.parametrize("layout", [LATENT, (8, 2, 128, True), (6, 2, 96, True)], ids=str)
def test_attention_sink_at_the_ends_of_its_range(ctx, W, layout, sink):
    value = {"lowest": torch.finfo(F32).min, "-inf": -np.inf, "high": 80.0}[sink]

    def spoil(c):
        c.sink[:] = value

    c = Case(18, *layout, [90, 0, 1], [1, 1, 1], 16, F32, spoil=spoil)
    c.check(W, ctx, sink=True)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True)], ids=str)
def test_attention_strides_streams_scratch_and_repeats(ctx, W, layout):
    heads, kvh, d, sep = layout
    c = Case(19, *layout, [301, 77, 1500], [2, 1, 1], 16, BF16)
    cache, cu = c.cache(W), dev(c.cu)
    lens, table = dev(np.array(c.lens, np.int32)), dev(c.table)
    a = W.kv_attention(ctx, cache, c.q, cu, lens, table)
    # head-major queries, outputs inside a wider tensor, garbage scratch, another stream
    q = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((c.q.shape[0], heads + 3, d + 16), 7.0, dtype=BF16, device="cuda")
    n = W.lib().wh_kv_attention_scratch_bytes(ctx.handle, __import__("ctypes").byref(cache.spec()),
                                              c.q.shape[0], heads, 3, 1)
    scratch = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = wide[:, 1:heads + 1, :d]
    b = W.kv_attention(ctx, cache, q, cu, lens, table, out=out, scratch=scratch, stream=side)
    side.synchronize()
    ctx.sync()
    assert torch.equal(a, b)
    assert (wide[:, 0] == 7).all() and (wide[:, heads + 1:] == 7).all() and (wide[..., d:] == 7).all()
    for _ in range(3):
        assert torch.equal(a, W.kv_attention(ctx, cache, c.q, cu, lens, table, scratch=scratch))


def test_attention_tokens_past_the_last_request_are_left_alone(ctx, W):
    c = Case(20, *LATENT, [100, 60], [1, 1], 16, BF16)
    q = torch.cat([c.q, c.q])
    out = torch.full_like(q, 3.0)
    W.kv_attention(ctx, c.cache(W), q, dev(c.cu), dev(np.array(c.lens, np.int32)), dev(c.table),
                   out=out)
    ctx.sync()
    assert (out[2:] == 3).all() and not (out[:2] == 3).all()


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True)], ids=str)
def test_attention_no_cu_q_means_one_query_each(ctx, W, layout):
    c = Case(21, *layout, [100, 0, 60], [1, 1, 1], 16, F32)
    args = (c.cache(W), c.q)
    lens, table = dev(np.array(c.lens, np.int32)), dev(c.table)
    a = W.kv_attention(ctx, *args, dev(c.cu), lens, table)
    b = W.kv_attention(ctx, *args, None, lens, table)
    ctx.sync()
    assert torch.equal(a, b)


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True), (6, 2, 96, True)], ids=str)
def test_attention_bad_blocks_and_lengths_are_recorded(ctx, W, layout):
    c = Case(22, *layout, [100, 60], [1, 1], 16, F32)
    cache, lens = c.cache(W), np.array(c.lens, np.int32)
    for bad in (-1, c.codes[0].shape[0], 1 << 30):
        table = c.table.copy()
        table[0, 2] = bad
        out = W.kv_attention(ctx, cache, c.q, None, dev(lens), dev(table))
        with pytest.raises(W.WohperError, match="DeviceArg"):
            ctx.sync()
        assert torch.isfinite(out).all()
    out = W.kv_attention(ctx, cache, c.q, None, dev(np.array([100, 5000], np.int32)), dev(c.table))
    with pytest.raises(W.WohperError, match="DeviceArg"):
        ctx.sync()
    assert torch.isfinite(out).all()
    W.kv_attention(ctx, cache, c.q, None, dev(np.array([100, -5], np.int32)), dev(c.table))
    with pytest.raises(W.WohperError, match="DeviceArg"):
        ctx.sync()
    ctx.sync()  # cleared


@pytest.mark.parametrize("layout", [LATENT, (28, 4, 128, True)], ids=str)
def test_attention_offsets_past_32_bits(ctx, W, layout):
    heads, kvh, d, sep = layout
    c = Case(23, *layout, [90, 300], [1, 2], 64, BF16)
    small = c.cache(W)
    blocks = c.codes[0].shape[0]
    total = (9 << 29) // (kvh * 64 * d // 2)  # 4.5 GiB of codes
    where = torch.arange(total - blocks, total, device="cuda")  # the last blocks of the pool

    def far(t, last):
        x = torch.empty(total, kvh, 64, last, dtype=torch.uint8, device="cuda")
        x[where] = t
        return x

    parts = [far(small.keys, d // 2), far(small.key_scales, d // 32)]
    if sep:
        parts += [far(small.values, d // 2), far(small.value_scales, d // 32)]
    table = np.where(c.table >= 0, c.table + (total - blocks), -1).astype(np.int32)
    lens = dev(np.array(c.lens, np.int32))
    a = W.kv_attention(ctx, small, c.q, dev(c.cu), lens, dev(c.table))
    big = W.PagedKvCache(*parts)
    b = W.kv_attention(ctx, big, c.q, dev(c.cu), lens, dev(table))
    assert torch.equal(a, b)
    slots = torch.tensor([(total - 1) * 64 + 63, (total - 1) * 64], device="cuda")
    x = torch.randn(2, kvh, d, device="cuda")
    W.kv_append(ctx, big, slots, x, x if sep else None)
    near = torch.tensor([(blocks - 1) * 64 + 63, (blocks - 1) * 64], device="cuda")
    W.kv_append(ctx, small, near, x, x if sep else None)
    ka, _ = W.kv_gather(ctx, big, slots)
    kb, _ = W.kv_gather(ctx, small, near)
    ctx.sync()
    assert torch.equal(ka, kb)


# ---------------------------------------------------------------------------
# append, gather
# ---------------------------------------------------------------------------
def edge_rows(rng, rows, kvh, d):
    """Rows whose blocks hold ties, range ends, zeros, subnormals and saturating values."""
    x = rng.standard_normal((rows, kvh, d)).astype(np.float32)
    x *= np.float32(2.0) ** rng.integers(-140, 120, (rows, kvh, 1)).astype(np.float32)
    ties = np.array([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5,
                     -5, -6, 0, -0.0, 0.2500001, 4.9999995], np.float32)
    x[0, 0, :32] = np.resize(ties, 32)
    x[1, 0, :32] = np.resize(ties, 32) * np.float32(2.0**-120)
    x[2, 0, :32] = 0.0
    x[3, 0, :32] = 3.0e38
    x[4, 0, :32] = np.float32(1e-45)
    x[5, 0, :32] = np.where(np.arange(32) == 7, 6.0000005, 0.3)
    return x


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("kvh,d,sep,page", [(1, 512, False, 64), (8, 128, True, 16), (3, 96, True, 7),
                                            (1, 32, False, 1)])
def test_append_codes_and_gather_values(ctx, W, dtype, kvh, d, sep, page):
    rng = np.random.default_rng(d)
    cache = W.PagedKvCache.empty(40, page, kvh, d, sep)
    rows = min(37, 40 * page - 3)
    k = dev(edge_rows(rng, rows, kvh, d)).to(dtype)
    v = dev(edge_rows(rng, rows, kvh, d)).to(dtype) if sep else None
    slots = torch.from_numpy(rng.permutation(40 * page)[:rows].astype(np.int64)).cuda()
    slots[10] = -1
    W.kv_append(ctx, cache, slots, k, v)
    ctx.sync()
    keep = np.arange(rows) != 10
    at = slots.cpu().numpy()[keep]
    every = torch.arange(40 * page, device="cuda")
    for x, codes, scales, got in zip((k, v), (cache.keys, cache.values),
                                     (cache.key_scales, cache.value_scales),
                                     W.kv_gather(ctx, cache, every)):
        if x is None:
            assert got is None
            continue
        c, s = R.quantise(x.double().cpu().numpy()[keep])
        want_c = np.zeros((40 * page, kvh, d // 2), np.uint8)
        want_s = np.zeros((40 * page, kvh, d // 32), np.uint8)
        want_c[at], want_s[at] = c, s
        got_c = codes.cpu().numpy().transpose(0, 2, 1, 3).reshape(40 * page, kvh, -1)
        got_s = scales.cpu().numpy().transpose(0, 2, 1, 3).reshape(40 * page, kvh, -1)
        np.testing.assert_array_equal(got_s, want_s)
        np.testing.assert_array_equal(got_c, want_c)
        values = R.values(want_c, want_s)
        np.testing.assert_array_equal(got.cpu().numpy(), values.astype(np.float32))
    for out_dtype in (BF16, F16):
        got, _ = W.kv_gather(ctx, cache, every, out_dtype)
        want = W.kv_gather(ctx, cache, every)[0].to(out_dtype)
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_append_rows_that_are_not_finite(ctx, W):
    cache = W.PagedKvCache.empty(1, 8, 1, 64)
    x = torch.randn(4, 1, 64, device="cuda")
    x[0, 0, 5] = float("nan")
    x[1, 0, 40] = float("inf")
    x[2, 0, 63] = -float("inf")
    slots = torch.arange(4, device="cuda")
    W.kv_append(ctx, cache, slots, x)
    got = W.kv_gather(ctx, cache, slots)[0].cpu().numpy()
    ctx.sync()
    nan = np.isnan(got).reshape(4, 2, 32)
    np.testing.assert_array_equal(nan.all(-1), [[True, False], [False, True], [False, True],
                                                [False, False]])
    np.testing.assert_array_equal(nan.any(-1), nan.all(-1))


def test_append_and_gather_strides_and_bad_slots(ctx, W):
    rng = np.random.default_rng(5)
    x = dev(rng.standard_normal((9, 4, 200)).astype(np.float32))
    k, v = x[:, 1:3, 8:136], x[:, 2:4, 40:168]
    pool = torch.zeros(6, 3, 2 * 5 * 64, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(6, 3, 16 * 3, dtype=torch.uint8, device="cuda")
    # layer 1 of a pool of 3 layers
    a = W.PagedKvCache(pool[:, 1].view(6, 2, 5, 64), scales[:, 1, :40].view(6, 2, 5, 4))
    slots = torch.tensor([0, 29, 7, -5, 12, 30, 1 << 40, 3, 15], device="cuda")
    W.kv_append(ctx, a, slots, k)
    with pytest.raises(W.WohperError, match="DeviceArg"):
        ctx.sync()
    got, _ = W.kv_gather(ctx, a, slots)
    with pytest.raises(W.WohperError, match="DeviceArg"):
        ctx.sync()
    want = R.values(*R.quantise(k.cpu().numpy()))
    want[[3, 5, 6]] = 0
    np.testing.assert_array_equal(got.cpu().numpy(), want.astype(np.float32))
    assert not pool[:, 0].any() and not pool[:, 2].any() and not scales[:, ::2].any()
    b = W.PagedKvCache.empty(6, 5, 2, 128, True)
    good = torch.arange(9, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    W.kv_append(ctx, b, good, k, v, stream=side)
    gk, gv = W.kv_gather(ctx, b, good, stream=side)
    side.synchronize()
    ctx.sync()
    np.testing.assert_array_equal(gk.cpu().numpy(), R.values(*R.quantise(k.cpu().numpy())).astype(np.float32))
    np.testing.assert_array_equal(gv.cpu().numpy(), R.values(*R.quantise(v.cpu().numpy())).astype(np.float32))


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------
def plan_case(seed, n, page, most, max_q, ending, spare=5):
    rng = np.random.default_rng(seed)
    old = rng.integers(0, most + 1, n)
    fin = rng.random(n) < ending
    q = np.where(fin, 0, rng.integers(0, max_q + 1, n))
    held, after = -(-old // page), -(-(old + q) // page)
    width = int(max(after.max(), held.max(), 1)) + 1
    blocks = int(held.sum() + (after - held).sum()) + spare
    order = rng.permutation(blocks).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    used = 0
    for r in range(n):
        table[r, :held[r]] = order[used:used + held[r]]
        used += int(held[r])
    free = np.full(blocks, -7, np.int32)
    free[:blocks - used] = order[used:]
    return old.astype(np.int32), q.astype(np.int32), fin, table, free, blocks - used


@pytest.mark.parametrize("n,page,most,max_q,ending", [
    (1, 64, 0, 1, 0), (1, 16, 100, 300, 0), (32, 64, 4096, 1, 0), (33, 1, 40, 3, 0.2),
    (700, 16, 500, 2, 0.1), (1025, 48, 300, 9, 0.5), (5000, 16, 64, 4, 0.1), (40, 16, 900, 700, 0.1),
    (8, 64, 128, 0, 0.9)])
def test_plan(ctx, W, n, page, most, max_q, ending):
    old, q, fin, table, free, top = plan_case(n + page, n, page, most, max_q, ending)
    t, f, tp, lens, cu, slots, pos, who = R.plan(page, old, q, fin, table, free, top)
    for pad in (0, 5):
        dt, df = dev(table), dev(free)
        p = W.kv_plan(ctx, page, dev(old), dev(q), dt, df, dev(np.array([top], np.int32)),
                      int(q.sum()) + pad, finished=dev(fin) if ending else None)
        ctx.sync()
        tail = [-1] * pad
        for got, want in ((dt, t), (df, f), (p.free_top, [tp]), (p.kv_lens, lens), (p.cu_q, cu),
                          (p.slots, slots + tail), (p.positions, pos + tail), (p.requests, who + tail)):
            np.testing.assert_array_equal(got.cpu().numpy(), np.array(want, got.cpu().numpy().dtype))


def test_plan_steps_on_another_stream_and_in_place_lengths(ctx, W):
    old, q, fin, table, free, top = plan_case(4, 9, 16, 30, 3, 0)
    side = torch.cuda.Stream()
    dt, df, tp = dev(table), dev(free), dev(np.array([top], np.int32))
    lens = dev(old)
    side.wait_stream(torch.cuda.current_stream())
    a = W.kv_plan(ctx, 16, lens, dev(q), dt, df, tp, int(q.sum()), stream=side)
    one = torch.ones(9, dtype=torch.int32, device="cuda")
    b = W.kv_plan(ctx, 16, a.kv_lens, torch.zeros_like(one), dt, df, a.free_top, 3, stream=side)
    side.synchronize()
    ctx.sync()
    assert torch.equal(a.kv_lens.cpu(), torch.from_numpy(old + q)) and torch.equal(a.kv_lens, b.kv_lens)
    assert int(b.cu_q[-1]) == 0 and (b.slots == -1).all() and torch.equal(a.free_top, b.free_top)


@pytest.mark.parametrize("what", ["blocks", "tokens", "length", "negative", "negative q", "ending q",
                                  "top", "overflow"])
@pytest.mark.parametrize("tokens", [40, 6000])
def test_plan_that_does_not_fit_changes_nothing(ctx, W, what, tokens):
    old, q, fin, table, free, top = plan_case(6, 12, 16, 200, 4, 0.3, spare=0)
    fin[0], fin[1], q[0] = True, False, 0
    old[0] = max(old[0], 20)
    q[2] = max(q[2], 1)
    if what == "blocks":
        q[1], tokens = 16 * (len(free) + 2), tokens + 16 * (len(free) + 2)
        table = np.concatenate([table, np.full((12, len(free) + 8), -1, np.int32)], 1)
    elif what == "tokens":
        tokens = int(q.sum()) - 1
    elif what == "length":
        old[1] = table.shape[1] * 16
        q[1] = 1
    elif what == "negative":
        old[3] = -1
    elif what == "negative q":
        q[3] = -1
    elif what == "ending q":
        q[0] = 1
    elif what == "top":
        top = len(free) + 1
    elif what == "overflow":
        top = len(free)
    dt, df = dev(table), dev(free)
    p = W.kv_plan(ctx, 16, dev(old), dev(q), dt, df, dev(np.array([top], np.int32)), tokens,
                  finished=dev(fin))
    with pytest.raises(W.WohperError, match="DeviceArg"):
        ctx.sync()
    np.testing.assert_array_equal(dt.cpu().numpy(), table)
    np.testing.assert_array_equal(df.cpu().numpy(), free)
    np.testing.assert_array_equal(p.kv_lens.cpu().numpy(), old)
    assert int(p.free_top) == top and not p.cu_q.any()
    assert (p.slots == -1).all() and (p.positions == -1).all() and (p.requests == -1).all()


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals(ctx, W):
    cache = W.PagedKvCache.empty(4, 16, 2, 128, True)
    lat = W.PagedKvCache.empty(4, 16, 1, 512)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, table = torch.ones(2, **i32), torch.zeros(2, 2, **i32)
    q = torch.zeros(2, 4, 128, device="cuda")
    slots = torch.arange(3, device="cuda")
    rows = torch.zeros(3, 2, 128, device="cuda")

    def refused(kind, fn, *a, **kw):
        with pytest.raises(W.WohperError) as e:
            fn(*a, **kw)
        assert e.value.kind == kind, e.value

    at = W.kv_attention
    refused("InvalidShape", at, ctx, cache, q[:, :3].contiguous(), None, lens, table)
    refused("InvalidShape", at, ctx, cache, q[..., :64], None, lens, table)
    refused("InvalidShape", at, ctx, cache, q[:1], None, lens, table)
    refused("InvalidShape", at, ctx, cache, q, lens, lens, table)
    refused("InvalidShape", at, ctx, cache, q, None, lens, table[:1])
    refused("InvalidShape", at, ctx, cache, q, None, lens, table, window=-1)
    refused("InvalidShape", at, ctx, cache, q, None, lens, table, first=-1)
    refused("InvalidShape", at, ctx, cache, q, None, lens, table, scale=float("nan"))
    refused("InvalidShape", at, ctx, cache, q, None, lens, table, sink=torch.zeros(3, device="cuda"))
    refused("InvalidShape", at, ctx, cache, q.transpose(1, 2).contiguous().transpose(1, 2), None, lens, table)
    refused("InvalidShape", at, ctx, cache, q, None, lens, table, out=torch.zeros(2, 4, 64, device="cuda"))
    refused("Unsupported", at, ctx, cache, q.double(), None, lens, table)
    refused("Unsupported", at, ctx, cache, q, None, lens.long(), table)
    refused("InvalidPointer", at, ctx, cache, q.cpu(), None, lens, table)
    refused("InvalidPointer", at, ctx, cache, torch.zeros(2 * 4 * 130, device="cuda")[1:1025].view(2, 4, 128), None,
            lens, table)
    refused("ScratchTooSmall", at, ctx, cache, q, None, lens, table, scratch=torch.zeros(1, dtype=torch.uint8, device="cuda"))
    refused("InvalidShape", W.kv_append, ctx, cache, slots, rows[:2], rows)
    refused("InvalidPointer", W.kv_append, ctx, cache, slots, rows)
    refused("InvalidPointer", W.kv_append, ctx, lat, slots, torch.zeros(3, 1, 512, device="cuda"),
            torch.zeros(3, 1, 512, device="cuda"))
    refused("Unsupported", W.kv_append, ctx, cache, slots, rows, rows.half())
    refused("Unsupported", W.kv_append, ctx, cache, slots.int(), rows, rows)
    refused("Unsupported", W.kv_gather, ctx, cache, slots, torch.float64)
    free, top = torch.zeros(4, **i32), torch.zeros(1, **i32)
    refused("InvalidShape", W.kv_plan, ctx, 16, lens, lens[:1], table, free, top, 2)
    refused("InvalidShape", W.kv_plan, ctx, 16, lens, lens, table[:1], free, top, 2)
    refused("InvalidShape", W.kv_plan, ctx, 16, lens, lens, table, free, top, -1)
    refused("EmptyShape", W.kv_plan, ctx, 0, lens, lens, table, free, top, 2)
    refused("Unsupported", W.kv_plan, ctx, 16, lens.long(), lens, table, free, top, 2)
    refused("Unsupported", W.kv_plan, ctx, 16, lens, lens, table, free, top, 2, finished=lens)
    refused("EmptyShape", at, ctx, cache, q[:0], torch.zeros(1, **i32), lens[:0], table[:0])
    assert at(ctx, cache, q[:0], torch.zeros(3, **i32), lens, table).shape == (0, 4, 128)
    W.kv_append(ctx, cache, slots[:0], rows[:0], rows[:0])
    assert W.kv_gather(ctx, cache, slots[:0])[0].shape == (0, 2, 128)
    ctx.sync()
