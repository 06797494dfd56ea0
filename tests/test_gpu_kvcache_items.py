"""The paged cache's attention where a CTA of the tensor-core kernel takes many short
items one after the other, and where items end early, begin in bad blocks or are
computed again.  Cases, plain 64-bit form and tolerances are those of
tests/test_gpu_kvcache.py."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_kvcache import BF16, F32, Case, ctx, dev, W  # noqa: F401 (fixtures)

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
