"""f32 attention over the paged 4-bit cache at lengths where one CTA adds up hundreds of
tiles: its error must not grow with the length.

The tensor cores drop what lies below an f32 sum's last bit, so a sum that runs through
many products shrinks: by half of the last place, 2^-24.5 of it, for each product of 16
rows.  Bounds on the signed error sum(err * sign(o)) / sum(|o|):
 - few query rows: a score is a sum of head_dim / 16 products, which moves a weight by
   that many times 2^-24.5 of the score; a group of 16 rows is one product of the weights'
   upper halves and one of the lower, added to f32 sums that round to nearest:
   2^-24.5 * (2 + head_dim / 16 * S), S the largest |score|;
 - the tensor-core kernel: besides that, 4 products a tile over at most 32 tiles before
   the sums are put aside: 2^-24.5 * (4 * 32 + head_dim / 16 * S).
The scores are kept below 1, and the number of outputs (10^5 and more) leaves nothing of
the errors without a sign."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def long_case(W, heads, kvh, d, sep, requests, rows, seed):
    """Random codes without signs, so that sums grow all the way, and ordinary scales for
    `requests` requests of `rows` rows, pages of 64."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = rows // 64
    blocks = requests * pages
    parts, u8 = [], dict(generator=g, device="cuda", dtype=torch.uint8)
    for _ in range(2 if sep else 1):
        parts.append(torch.randint(0, 256, (blocks, kvh, 64, d // 2), **u8) & 0x77)
        parts.append(torch.randint(124, 127, (blocks, kvh, 64, d // 32), **u8))
    table = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32).view(requests, pages)
    q = torch.randn(requests, heads, d, generator=g, device="cuda") * 0.02
    lens = torch.full((requests,), rows, dtype=torch.int32, device="cuda")
    return W.PagedKvCache(*parts), q, lens, table


def real(codes, scales):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = grid[c & 7] * (1 - 2 * (c >> 3))
    return (v.unflatten(-1, (-1, 32)) * 2.0 ** (scales.double() - 127)[..., None]).flatten(-2)


def exact(cache, q, table, r):
    """(outputs [heads, d] of request r in 64 bits, its largest |score|)"""
    heads, d = q.shape[1:]
    at = table[r].long()
    k = real(cache.keys[at], cache.key_scales[at]).transpose(0, 1).flatten(1, 2)  # [kvh, rows, d]
    v = k if cache.values is None else real(cache.values[at], cache.value_scales[at]).transpose(0, 1).flatten(1, 2)
    s = q[r].double().view(cache.kv_heads, -1, d) @ k.transpose(1, 2) * d**-0.5
    return (torch.softmax(s, -1) @ v).view(heads, d), float(s.abs().max())


@pytest.mark.parametrize("name,layout,requests,rows", [
    ("few", (8, 8, 128, True), 64, 32768), ("few", (32, 8, 64, False), 64, 32768), ("few", (16, 2, 256, False), 64, 65536),
    ("tc", (64, 1, 512, False), 48, 49152), ("tc", (64, 1, 128, True), 48, 49152), ("tc", (64, 2, 64, False), 64, 32768)],
    ids=str)
def test_f32_sums_do_not_shrink_with_the_length(name, layout, requests, rows):
    import wohper_b200 as W

    ctx = W.Context(0)
    cache, q, lens, table = long_case(W, *layout, requests, rows, 1)
    got = W.kv_attention(ctx, cache, q, None, lens, table)
    ctx.sync()
    err = top = 0.0
    largest = 0.0
    for r in range(0, requests, 5):
        want, s = exact(cache, q, table, r)
        err += float(((got[r].double() - want) * want.sign()).sum())
        top += float(want.abs().sum())
        largest = max(largest, s)
    assert largest < 1
    products = layout[2] / 16 * largest + (4 * 32 if name == "tc" else 2)
    assert abs(err / top) <= 2.0**-24.5 * products, (err / top, 2.0**-24.5 * products)
    ctx.close()


@pytest.mark.parametrize("layout", [(8, 2, 128, True), (64, 1, 128, True), (64, 2, 64, True), (40, 1, 512, True),
                                    (6, 2, 96, True)], ids=str)
@pytest.mark.parametrize("wide", [20, 26, 30])
def test_f32_weights_far_below_the_largest_still_count(layout, wide):
    # One row with a weight of 1 and the value 0 among rows whose weights are all
    # e^-(0.75 wide) = 2^-21.6, 2^-28.1, 2^-32.5: the output is theirs alone.  A weight is the sum of two
    # f16, the lower one held 2^11 times larger: at 2^9 times the weight the upper one is
    # rounded to 2^-24 at the finest and the lower one to 2^-35, so that a weight of
    # 2^-32.5 is off by at most 2^-36 of 2^-23.5, or 2^-12 of itself; the score's error
    # (tests/test_gpu_kvcache.py) comes on top.
    import numpy as np

    import wohper_b200 as W
    from tests import kv_reference as R
    from tests.test_gpu_kvcache import F32, Case, dev

    def spoil(c):
        peak = np.zeros(layout[2])
        peak[:wide] = 0.75
        c.scales[0][:] = 0  # keys of zeros, but for one
        b = c.table[0, 60 // 16]
        c.codes[0][b, :, 60 % 16], c.scales[0][b, :, 60 % 16] = R.quantise(peak)
        c.codes[1] &= 0x77
        c.scales[1][b, :, 60 % 16] = 0
        c.q = torch.ones_like(c.q)

    ctx = W.Context(0)
    c = Case(36, *layout, [900], [1], 16, F32, spoil=spoil)
    got = W.kv_attention(ctx, c.cache(W), c.q, None, dev(np.array(c.lens, np.int32)), dev(c.table), scale=1.0)
    ctx.sync()
    want, smax, _ = c.want(1.0)
    assert (want > 0).all()
    ratio = np.abs(got.double().cpu().numpy() / want - 1)
    assert (ratio <= 2.0**-12 + 2.0**-22 * (16 + 8 * smax.max())).all(), ratio.max()
    ctx.close()
