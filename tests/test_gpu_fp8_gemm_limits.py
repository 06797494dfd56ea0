"""The FP8 product's limits, asked for with pointers that are never read."""
from __future__ import annotations

import pytest

from tests.test_gpu_fp8_gemm import W, ctx  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,tokens", [((1 << 30) + 16, 16, 1), (16, (1 << 30) + 16, 1), (16, 16, (1 << 30) + 1),
                                              ((1 << 31) - 16, 16, 1), (16, (1 << 31) - 16, 1), (16, 16, (1 << 31) - 1)])
def test_sizes_past_the_limit_are_refused(ctx, W, rows, cols, tokens):  # noqa: F811
    p = torch.zeros(256, dtype=torch.uint8, device="cuda").data_ptr()
    status = W.lib().wh_fp8_gemm(ctx.handle, p, p, rows, cols, -(-rows // 128), -(-cols // 128), p, 1, tokens, cols, p, 1, rows, 64,
                                 p, W.lib().wh_fp8_gemm_scratch_bytes(cols, tokens), 0)
    assert status == 10  # WH_ERR_UNSUPPORTED
    ctx.sync()
