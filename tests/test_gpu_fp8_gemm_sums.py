"""How much the FP8 product's 16-bit outputs lose downwards over very long rows.

The tensor core cuts its running sum off with each instruction of 32 columns: 2^-22 of the sum
at most is allowed for it, as in test_gpu_fp8_gemm.py.  With positive terms the running sum grows
evenly, so n instructions lose at most n / 2 * 2^-22 of a sum: 256 (8192 columns, after
which the sum is added in f32) 2^-15, and 32 (1024 columns, an f32 output's) 2^-18.  The mean over
many outputs shows it, since roundings to f16, uniform within 2^-11 of the value, average out: over N
outputs to 2^-11 / sqrt(3 N), of which 5 are allowed.  An f32 output's own additions, one
for each 1024 columns of a CTA, round to nearest, 2^-24 of the running sum each.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_fp8_gemm import BF16, F16, F32, W, ctx  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("long", [32768, 393216])  # columns of each of the eight CTAs that share a row
def test_sums_of_16_bit_outputs_are_added_after_8192_columns(ctx, W, long):  # noqa: F811
    rows, tokens, cols = 128, 64, 8 * long
    g = torch.Generator(device="cuda").manual_seed(11)
    w = torch.randint(0, 127, (rows, cols), generator=g, device="cuda", dtype=torch.uint8)  # positive, no NaN
    s = torch.full((1, cols // 128), 127 - 18, dtype=torch.uint8, device="cuda")
    x = torch.empty(tokens, cols, dtype=BF16, device="cuda")
    for t in range(tokens):  # another size for each token, so that roundings differ
        x[t] = (torch.rand(cols, generator=g, device="cuda") + 0.01) * float(np.exp2(t / tokens))
    near = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, out_dtype=F32).double()
    half = W.gemm_fp8_e4m3_ue8m0(ctx, w, s, x, out_dtype=F16)
    ctx.sync()
    assert half.isfinite().all()
    lost = float(((half.double() - near) / near).mean())
    rounding = 5 * 2.0**-11 / (3 * rows * tokens) ** 0.5
    assert -(2.0**-15 + rounding) <= lost <= 2.0**-18 + long / 1024 / 2 * 2.0**-24 + rounding, lost
