"""The example server loop on the paged 4-bit cache: lengths, block accounting and
one decode step's outputs against the plain 64-bit form."""
from __future__ import annotations

import numpy as np
import pytest

from tests import kv_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_example_runs_and_accounts_for_every_block():
    from examples import paged_serving

    r = paged_serving.main(steps=70)
    prompts = [70, 1, 200, 33, 128, 5, 64, 150]
    assert r["lens"] == [p + 70 for p in prompts]
    assert r["after"] == [0 if i in (1, 4) else p + 71 for i, p in enumerate(prompts)]
    assert r["free"] + r["held"] == r["blocks"] and r["finite"]


def test_captured_step_equals_the_plain_form():
    import wohper_b200 as W
    from examples.paged_serving import PagedServer

    ctx = W.Context(0)
    s = PagedServer(ctx, slots=3, layers=2, blocks=20, page=16, window=40, first=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    prompts = [90, 7, 50]

    def inputs(n):
        return ([torch.randn(n, s.d, generator=g, device="cuda") for _ in range(2)],
                [torch.randn(n, s.heads, s.d, generator=g, device="cuda").bfloat16() for _ in range(2)])

    s.step(torch.tensor(prompts, dtype=torch.int32, device="cuda"), *inputs(sum(prompts)))
    graph, q_lens, rows, queries, out = s.capture(3)
    q_lens.fill_(1)
    for _ in range(3):
        r, q = inputs(3)
        for a, b in zip(rows + queries, r + q):
            a.copy_(b)
        graph.replay()
    ctx.sync()
    lens = [p + 3 for p in prompts]
    assert s.lens.tolist() == lens
    cache = s.caches[1]
    values = R.values(cache.keys.cpu().numpy(), cache.key_scales.cpu().numpy())
    want, smax, vmax = R.attend(queries[1].double().cpu().numpy(), values, values, [0, 1, 2, 3], lens,
                                s.table.cpu().numpy(), 16, s.d**-0.5, 40, 3, np.zeros(64))
    err = np.abs(out.double().cpu().numpy() - want)
    # weights of 11 bits and a bf16 output, beside the f32 score's error (tests/test_gpu_kvcache.py)
    tol = (vmax * (2.0**-11 + 2.0**-22 * (16 + 8 * smax)))[..., None] + 2.0**-8 * np.abs(want) + 2.0**-25
    assert (err <= tol).all(), float((err / tol).max())
    graph.reset()
    ctx.close()
