"""The FP8 product of one and two tokens, quantised inside, where a CTA has more K tiles
than its warps fill once: against 64-bit products (tolerances of test_gpu_fp8_gemm.py),
and the same bits call after call.  What the warps wait for is run through on the CPU
(test_fp8_gemm_steps.py)."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_fp8_gemm import BF16, F16, F32, W, check, ctx, inputs, quantised, weight  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def again_and_again(ctx, W, rows, cols, tokens, dtype, out_dtype):  # noqa: F811
    rng = np.random.default_rng(cols + tokens)
    block = (32, 64, 128)[(cols // 16 + tokens) % 3]
    w, s, real = weight(rng, rows, cols)
    x = inputs(rng, tokens, cols, dtype)
    y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, block, out_dtype)
    ctx.sync()
    check(y, real, quantised(x, block), out_dtype)
    for _ in range(30):
        z = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, block, out_dtype)
        assert torch.equal(y, z)
    ctx.sync()


@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, BF16), (F16, F16), (F16, F32)], ids=str)
@pytest.mark.parametrize("tokens", [1, 2])
@pytest.mark.parametrize("tiles", [8, 9, 10, 12, 13, 16, 17, 18, 24, 25, 33, 96])
def test_many_k_tiles_a_cta(ctx, W, tiles, tokens, dtype, out_dtype):  # noqa: F811
    # two rows of tiles, each by a cluster of eight; the last K tile is ragged
    again_and_again(ctx, W, 130, 1024 * tiles - 16 * (tiles % 8), tokens, dtype, out_dtype)


@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, BF16), (F16, F16)], ids=str)
@pytest.mark.parametrize("tokens", [1, 2])
def test_rows_that_leave_no_shares(ctx, W, tokens, dtype, out_dtype):  # noqa: F811
    again_and_again(ctx, W, 20000, 1168, tokens, dtype, out_dtype)
