"""The FP8 product writes its columns of a wider output and nothing beside them."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_fp8_gemm import BF16, F16, F32, W, check, ctx, inputs, quantised, weight  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("tokens", [1, 2, 5, 43, 130, 580])
@pytest.mark.parametrize("rows,cols", [(1, 48), (29, 288), (97, 224), (100, 224), (127, 144), (131, 144), (252, 208), (1287, 144),
                                       (4421, 48)])
def test_rows_that_end_between_16_bytes(ctx, W, rows, cols, tokens, out_dtype):  # noqa: F811
    # a row of the output holds `rows` columns of the product and others behind them, and starts on 16 bytes
    rng = np.random.default_rng(rows + tokens)
    w, s, real = weight(rng, rows, cols)
    x = inputs(rng, tokens, cols, BF16)
    for more in (0, 8):
        out = torch.full((tokens, -(-rows // 8) * 8 + more), 7.0, dtype=out_dtype, device="cuda")
        y = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, out=out[:, :rows])
        ctx.sync()
        assert (out[:, rows:] == 7).all()
        check(y, real, quantised(x, 64), out_dtype)


@pytest.mark.parametrize("out_dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("tokens", [40, 300])
def test_products_side_by_side(ctx, W, tokens, out_dtype):  # noqa: F811
    # each begins on 16 bytes, the last column of one beside the first of the next
    rng = np.random.default_rng(tokens)
    step = 16 // torch.empty(0, dtype=out_dtype).element_size()
    x = inputs(rng, tokens, 144, F32)
    out = torch.full((tokens, 1024), 7.0, dtype=out_dtype, device="cuda")
    parts, at = [], 0
    for rows in (21, 139, 3, 130, 257, 1):
        parts.append((at, rows, weight(rng, rows, 144)))
        at += -(-rows // step) * step
    for order in (parts, parts[::-1]):  # either neighbour first
        out.fill_(7.0)
        for a, rows, (w, s, _) in order:
            W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, out=out[:, a:a + rows])
        ctx.sync()
        mine = torch.zeros(1024, dtype=torch.bool, device="cuda")
        for a, rows, (_, _, real) in parts:
            check(out[:, a:a + rows], real, quantised(x, 64), out_dtype)
            mine[a:a + rows] = True
        assert (out[:, ~mine] == 7).all()
