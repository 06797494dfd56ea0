"""The FP8 product of many tokens on the GPU against 64-bit products of the same
operands (the oracle's act quant and FP8 values).

Tolerance, with A = sum |w x| of an output.  The products are exact.  A tensor-core
instruction adds 32 of them to the running sum; aligned to the largest of them and cut
off, that loses at most a few 2^-24 of A: 2^-22 A is allowed for each of the
instructions, of which at most 32 follow one another before the sum is added in f32
for an f32 output (each such addition: 2^-24 A), all of cols / 32 for a 16-bit one.
16-bit outputs add their rounding, 2^-8 (bf16) or 2^-11 (f16) of the value, and
2^-25 for f16's subnormals.
"""
from __future__ import annotations

import numpy as np
import pytest

import oracle as O

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


def e4m3(b):
    b = b.astype(np.int64)
    e, m = (b & 127) >> 3, (b & 7).astype(np.float64)
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7.0), m / 8 * 2.0**-6)
    return np.where(b & 128, -v, v)


def weight(rng, rows, cols, lo=110, hi=120):
    w = rng.integers(0, 256, (rows, cols)).astype(np.uint8)
    w[(w & 127) == 127] = 0x30  # no NaN
    s = rng.integers(lo, hi, (-(-rows // 128), -(-cols // 128))).astype(np.uint8)
    real = e4m3(w) * np.repeat(np.repeat(2.0 ** (s - 127.0), 128, 0)[:rows], 128, 1)[:, :cols]
    return torch.from_numpy(w).cuda(), torch.from_numpy(s).cuda(), real


def quantised(x, block):
    """The oracle's act quant of each row's blocks, the last one ragged."""
    x = x.float().cpu().numpy()
    out = x.copy()
    for t in range(x.shape[0]):
        for c in range(0, x.shape[1], block):
            part = np.ascontiguousarray(x[t, c:c + block])
            out[t, c:c + block] = O.act_quant(part, part.size)
    return out.astype(np.float64)


def check(got, real, xq, dtype):
    want, size = xq @ real.T, np.abs(xq) @ np.abs(real).T
    cols = real.shape[1]
    steps = min(32, cols / 32 + 1) + cols / 1024 / 4 if dtype == F32 else cols / 32 + 1
    tol = size * 2.0**-22 * steps + UNIT[dtype] * np.abs(want) + (2.0**-25 if dtype == F16 else 0.0)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())


def inputs(rng, tokens, cols, dtype):
    x = rng.standard_normal((tokens, cols)) * np.exp(rng.standard_normal((tokens, 1)))
    x[:, rng.random(cols) < 0.02] *= 8
    return torch.from_numpy(x.astype(np.float32)).cuda().to(dtype)


@pytest.mark.parametrize("rows,cols", [(1, 16), (128, 128), (129, 144), (1000, 1360), (384, 2064), (257, 4096)])
@pytest.mark.parametrize("tokens", [1, 16, 17, 33, 64, 65, 128, 129, 256, 257, 300])
def test_sizes(ctx, W, rows, cols, tokens):
    rng = np.random.default_rng(rows + cols + tokens)
    dtype, block = ((F32, 64), (BF16, 128), (F16, 32))[(rows + tokens) % 3]
    w, s, real = weight(rng, rows, cols)
    x = inputs(rng, tokens, cols, dtype)
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, act_quant_block=block)
    ctx.sync()
    assert y.shape == (tokens, rows) and y.dtype is dtype
    check(y, real, quantised(x, block), dtype)


@pytest.mark.parametrize("rows,cols,tokens", [(100, 20496, 3), (100, 20496, 30), (100, 20496, 140), (19200, 2560, 3),
                                              (19200, 2560, 30), (19200, 2560, 140), (640, 12288, 3), (640, 12288, 140),
                                              (1300, 1168, 4500), (2048, 512, 5000), (300, 144, 20000),
                                              (4096, 256, 8192)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_long_sums(ctx, W, rows, cols, tokens, dtype):
    # many sums of 1024 columns to a tile, alone in it and shared by a cluster
    rng = np.random.default_rng(rows)
    w, s, real = weight(rng, rows, cols)
    x = inputs(rng, tokens, cols, dtype)
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x)
    ctx.sync()
    check(y, real, quantised(x, 64), dtype)


@pytest.mark.parametrize("rows,cols", [(1, 16), (129, 144), (4096, 2064), (300, 20496), (19200, 2560)])
@pytest.mark.parametrize("tokens", [1, 2])
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (F32, F16), (BF16, BF16), (F16, F32)], ids=str)
def test_one_and_two_tokens(ctx, W, rows, cols, tokens, dtype, out_dtype):
    # quantised inside the product; 19200 rows leave no CTAs to share a tile's K
    rng = np.random.default_rng(rows)
    block = (32, 64, 128)[(rows + tokens) % 3]
    w, s, real = weight(rng, rows, cols)
    wide = torch.zeros(tokens, 2 * cols, dtype=dtype, device="cuda")
    x = wide[:, cols:]
    x.copy_(inputs(rng, tokens, cols, dtype))
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, block, out_dtype)
    z = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x.contiguous(), block, out_dtype)
    ctx.sync()
    check(y, real, quantised(x, block), out_dtype)
    assert torch.equal(y, z)


@pytest.mark.parametrize("tokens", [1, 2])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_one_of_two_tokens_that_is_not_finite(ctx, W, tokens, bad):
    rng = np.random.default_rng(8)
    w, s, real = weight(rng, 300, 1040)
    w[w == 0] = 1
    x = inputs(rng, tokens, 1040, F32)
    clean = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x)
    for t in range(tokens):
        z = x.clone()
        z[t, 1039] = bad
        y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, z)
        keep = torch.arange(tokens, device="cuda") != t
        assert y[t].isnan().all() and torch.equal(y[keep], clean[keep])
    ctx.sync()


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("tokens", [1, 40])
def test_very_long_rows(ctx, W, tokens, out_dtype):
    # positive terms, whose sums a tensor core rounds down; added in f32 after 1024 columns
    # for f32 and 32768 for 16-bit outputs: 2^-24 of the sum for each instruction before
    rng = np.random.default_rng(9)
    w, s, _ = weight(rng, 130, 98320)
    w &= 127
    real = e4m3(w.cpu().numpy()) * np.repeat(np.repeat(2.0 ** (s.cpu().numpy() - 127.0), 128, 0)[:130], 128, 1)[:, :98320]
    x = inputs(rng, tokens, 98320, F32).abs() * 2.0**-10
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, 64, out_dtype)
    ctx.sync()
    want = quantised(x, 64) @ real.T
    steps = (32 if out_dtype == F32 else 1024) + 98320 / 1024 / 4
    err = np.abs(y.double().cpu().numpy() - want)
    assert (err <= np.abs(want) * (2.0**-22 * steps + UNIT[out_dtype])).all(), float((err / want).max())


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("out_dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("tokens", [5, 200])
@pytest.mark.parametrize("block", [32, 64, 128])
def test_types(ctx, W, dtype, out_dtype, tokens, block):
    rng = np.random.default_rng(tokens + block)
    w, s, real = weight(rng, 300, 1040)
    x = inputs(rng, tokens, 1040, dtype)
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, block, out_dtype)
    ctx.sync()
    check(y, real, quantised(x, block), out_dtype)


@pytest.mark.parametrize("tokens", [3, 150])
def test_equals_the_gemv_on_the_same_operands(ctx, W, tokens):
    # the GEMV's sums are f32 chains of 16 lanes: at most cols / 16 roundings of 2^-24 A each
    rng = np.random.default_rng(1)
    w, s, real = weight(rng, 256, 2048)
    x = inputs(rng, tokens, 2048, F32)
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x)
    z = W.gemv_fp8_e4m3_ue8m0_rows_multi(ctx, w, s, x[:32].contiguous(), 0, 256, act_quant_block=64)
    ctx.sync()
    size = np.abs(quantised(x[:32], 64)) @ np.abs(real).T
    err = np.abs(y[:32].double().cpu().numpy() - z.double().cpu().numpy())
    assert (err <= size * (2.0**-22 * 34 + 2.0**-24 * 128)).all()


@pytest.mark.parametrize("lo,hi", [(1, 40), (60, 200), (0, 1)])
@pytest.mark.parametrize("tokens", [4, 140])
def test_scale_bytes_over_the_whole_range(ctx, W, lo, hi, tokens):
    # a scale byte 0 is 2^-127; sums stay inside f32
    rng = np.random.default_rng(lo + tokens)
    w, s, real = weight(rng, 256, 512, lo, hi)
    x = inputs(rng, tokens, 512, F32) * (2.0**20 if hi < 100 else 2.0**-20)
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x)
    ctx.sync()
    xq = quantised(x, 64)
    want, size = xq @ real.T, np.abs(xq) @ np.abs(real).T
    err = np.abs(y.double().cpu().numpy() - want)
    # f32's subnormals: half of 2^-149 for each addition
    assert (err <= size * 2.0**-22 * 18 + 2.0**-149 * 20).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("tokens", [1, 2, 50])
def test_codes_are_the_act_quants_at_ties_and_beside_them(ctx, W, dtype, block, tokens):
    # a weight of ones on its diagonal gives the quantised tokens back, exactly
    grid = e4m3(np.arange(127, dtype=np.uint8))
    near = np.concatenate([grid, (grid[1:] + grid[:-1]) / 2]).astype(np.float32)
    bits = near[near > 0].view(np.int32)
    near = np.concatenate([(bits + d).astype(np.int32).view(np.float32) for d in range(-3, 4)] + [np.zeros(9, np.float32)])
    rng = np.random.default_rng(block + tokens)
    n = 1040
    x = rng.choice(near, (tokens, n)) * rng.choice([-1, 1], (tokens, n)).astype(np.float32)
    x[:, ::block] = 448 * rng.choice([-1, 1], x[:, ::block].shape)  # the block's scale is the token's
    x *= 2.0 ** rng.integers(-6, 7, (tokens, 1)).astype(np.float32)
    x = torch.from_numpy(x).cuda().to(dtype)
    w = torch.zeros(n, n, dtype=torch.uint8, device="cuda")
    w.fill_diagonal_(0x38)
    s = torch.full((9, 9), 127, dtype=torch.uint8, device="cuda")
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, block, F32)
    ctx.sync()
    assert (y.double().cpu().numpy() == quantised(x, block)).all()


@pytest.mark.parametrize("tokens", [2, 2000])
def test_scales_around_their_thresholds(ctx, W, tokens):
    # the largest value of each block lies a few last places from where its scale doubles
    rng = np.random.default_rng(tokens)
    n = 1024
    x = rng.standard_normal((tokens, n // 64, 64)).astype(np.float32)
    e = rng.integers(-22, 119, (tokens, n // 64))
    step = np.concatenate([np.arange(-4, 40), 2 ** np.arange(5, 24), -(2 ** np.arange(2, 23))])
    top = (np.float32(448) * 2.0 ** e.astype(np.float32)).astype(np.float32).view(np.int32) + rng.choice(step, e.shape)
    top = np.maximum(top.astype(np.int32).view(np.float32), np.float32(1e-5))
    x *= top[..., None] / 8
    x[:, :, 5] = top
    x = torch.from_numpy(x.reshape(tokens, n)).cuda()
    x = torch.where(x.abs() > torch.from_numpy(top).cuda().repeat_interleave(64, 1), 0.0, x)
    w = torch.zeros(n, n, dtype=torch.uint8, device="cuda")
    w.fill_diagonal_(0x38)
    s = torch.full((8, 8), 127, dtype=torch.uint8, device="cuda")
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x)
    ctx.sync()
    assert (y.double().cpu().numpy() == quantised(x, 64)).all()


def test_tiny_huge_and_zero_tokens(ctx, W):
    rng = np.random.default_rng(2)
    w, s, real = weight(rng, 130, 272)
    x = inputs(rng, 6, 272, F32)
    x[0] = 0.0
    x[1] *= 1e-30
    x[2] *= 1e25
    x[3, :128] = 0.0
    x[4, ::2] = -0.0
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x)
    ctx.sync()
    check(y, real, quantised(x, 64), F32)
    assert (y[0] == 0).all() and not y[0].signbit().any()


@pytest.mark.parametrize("tokens", [8, 200])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_token_that_is_not_finite_spoils_only_itself(ctx, W, tokens, bad):
    rng = np.random.default_rng(3)
    w, s, real = weight(rng, 200, 512)
    w[w == 0] = 1  # a weight 0 times NaN is NaN as well; without zeros every row shows it
    x = inputs(rng, tokens, 512, BF16)
    clean = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x)
    x[5, 77] = bad
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x)
    ctx.sync()
    assert y[5].isnan().all()
    keep = torch.arange(tokens, device="cuda") != 5
    assert torch.equal(y[keep], clean[keep]) and y[keep].isfinite().all()


def test_nan_weights_and_scales_reach_their_rows(ctx, W):
    rng = np.random.default_rng(4)
    w, s, _ = weight(rng, 300, 512)
    x = inputs(rng, 9, 512, F32)
    clean = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x)
    w[7, 100], w[299, 500] = 0x7F, 0xFF
    s[1, 2] = 255
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x)
    ctx.sync()
    bad = torch.zeros(300, dtype=torch.bool, device="cuda")
    bad[7] = bad[299] = True
    bad[128:256] = True
    assert y[:, bad].isnan().all() and torch.equal(y[:, ~bad], clean[:, ~bad])


@pytest.mark.parametrize("tokens", [1, 7, 130, 300])
def test_strides_streams_scratch_graphs_and_repeats(ctx, W, tokens):
    rng = np.random.default_rng(5)
    w, s, _ = weight(rng, 272, 528)
    x = inputs(rng, tokens, 528, BF16)
    a = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, 32)
    wide = torch.zeros(tokens, 3 * 528 + 8, dtype=BF16, device="cuda")
    wide[:, 528:1056] = x
    out = torch.full((tokens, 301), 7.0, dtype=BF16, device="cuda")
    scratch = torch.full((W.lib().wh_fp8_gemm_scratch_bytes(528, tokens),), 255, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, wide[:, 528:1056], 32, out=out[:, 11:283], scratch=scratch, stream=side)
    torch.cuda.synchronize()
    assert got.data_ptr() == out[:, 11:283].data_ptr() and torch.equal(got, a)
    assert (out[:, :11] == 7).all() and (out[:, 283:] == 7).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, 32)
    for _ in range(3):
        y.zero_()
        g.replay()
        assert torch.equal(y, a)
    ctx.sync()
    g.reset()


def test_a_group_of_a_wider_projection(ctx, W):
    # the grouped low-rank projection: each group's rows on its own slice of the input
    rng = np.random.default_rng(6)
    w, s, _ = weight(rng, 512, 256)
    x = inputs(rng, 40, 1024, F32)
    y = torch.empty(40, 512, device="cuda")
    for g in range(4):
        W.gemm_fp8_e4m3_ue8m0(ctx, w[128 * g:128 * g + 128], s[g:g + 1], x[:, 256 * g:256 * g + 256], out=y[:, 128 * g:128 * g + 128])
    for t in (0, 39):
        one = W.gemv_fp8_e4m3_ue8m0_grouped(ctx, w, s, x[t].contiguous(), 128, 256, act_quant_block=64)
        assert torch.allclose(y[t], one, rtol=1e-4, atol=1e-3 * float(one.abs().max()))
    ctx.sync()


def refused(W, kind, *a, **kw):
    with pytest.raises(W.WohperError) as e:
        W.gemm_fp8_e4m3_ue8m0(*a, **kw)
    assert e.value.kind == kind, e.value


def test_refusals_and_no_tokens(ctx, W):
    rng = np.random.default_rng(7)
    w, s, _ = weight(rng, 130, 272)
    x = inputs(rng, 4, 272, F32)
    refused(W, "Unsupported", ctx, w[:, :264].contiguous(), s, x[:, :264])
    refused(W, "InvalidShape", ctx, w[:, :256], s[:, :2].contiguous(), x[:, :256])  # a weight that is not dense
    refused(W, "InvalidShape", ctx, w, s[:1], x)
    refused(W, "InvalidShape", ctx, w, s, x[:, :256])
    refused(W, "InvalidShape", ctx, w, s, x.t().contiguous().t())
    refused(W, "InvalidShape", ctx, w, s, x[:1].expand(4, 272))
    refused(W, "InvalidPointer", ctx, w, s, torch.cat([x, x], 1)[:, 1:273])
    refused(W, "InvalidPointer", ctx, w, s, x.cpu())
    refused(W, "InvalidPointer", ctx, w, s.cpu(), x)
    refused(W, "Unsupported", ctx, w, s, x.double())
    refused(W, "Unsupported", ctx, w, s, x, out_dtype=torch.float64)
    refused(W, "Unsupported", ctx, w, s.int(), x)
    refused(W, "Unsupported", ctx, w, s, x, act_quant_block=48)
    refused(W, "Unsupported", ctx, w, s, x, act_quant_block=0)
    refused(W, "InvalidShape", ctx, w, s, x, out=torch.empty(4, 131, device="cuda"))
    refused(W, "InvalidShape", ctx, w, s, x, out=torch.empty(130, device="cuda").expand(4, 130))
    refused(W, "Unsupported", ctx, w, s, x, out_dtype=BF16, out=torch.empty(4, 130, device="cuda"))
    refused(W, "ScratchTooSmall", ctx, w, s, x.repeat(3, 1), scratch=torch.empty(100, dtype=torch.uint8, device="cuda"))
    assert W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x[:0]).shape == (0, 130)
    ctx.sync()
