"""CPU checks of the paged 4-bit cache: what its pool refuses, and the plain
64-bit forms (tests/kv_reference.py) against their own definitions."""
from __future__ import annotations

import numpy as np
import pytest

from tests import kv_reference as R

torch = pytest.importorskip("torch")


def _pool(b=3, h=2, p=5, d=64, sep=False):
    def z(last):
        return torch.zeros(b, h, p, last, dtype=torch.uint8)

    return [z(d // 2), z(d // 32)] + ([z(d // 2), z(d // 32)] if sep else [])


def test_pool_shapes_and_strides():
    import wohper_b200 as W

    c = W.PagedKvCache(*_pool(sep=True))
    assert (c.blocks, c.page, c.kv_heads, c.head_dim) == (3, 5, 2, 64)
    assert c.spec().block_stride == 2 * 5 * 32 and c.spec().scale_block_stride == 2 * 5 * 2
    wide = torch.zeros(3, 4, 2, 5, 32, dtype=torch.uint8)
    c = W.PagedKvCache(wide[:, 1], _pool()[1])
    assert c.spec().block_stride == 4 * 2 * 5 * 32
    e = W.PagedKvCache.empty(2, 4, 1, 96, device="cpu")
    assert e.head_dim == 96 and e.values is None


def test_pool_refusals():
    import wohper_b200 as W

    def refused(kind, *a, **kw):
        with pytest.raises(W.WohperError) as e:
            W.PagedKvCache(*a, **kw)
        assert e.value.kind == kind

    k, s, v, vs = _pool(sep=True)
    refused("InvalidShape", k[0], s)
    refused("InvalidShape", k, s[..., :1])
    refused("InvalidShape", k[..., :24], s)
    refused("InvalidShape", k.transpose(1, 2).contiguous().transpose(1, 2), s)
    refused("InvalidShape", k, s, v[:, :1], vs)
    refused("InvalidPointer", k, s, v)
    refused("Unsupported", k.int(), s)
    wide = torch.zeros(3, 4, 2, 5, 32, dtype=torch.uint8)
    refused("InvalidShape", wide[:, 0], s, v, vs)
    with pytest.raises(W.WohperError):
        W.PagedKvCache.empty(1, 1, 1, 48, device="cpu")


def test_reference_quantiser_is_nearest_on_its_grid():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 64)) * 2.0 ** rng.integers(-40, 40, (40, 1))
    codes, scales = R.quantise(x)
    got = R.values(codes, scales)
    unit = np.repeat(2.0 ** (scales.astype(float) - 127), 32, -1).reshape(x.shape)
    top = np.abs(x).reshape(40, 2, 32).max(-1)
    assert (top <= 6 * unit.reshape(40, 2, 32)[..., 0]).all()
    assert (top > 3 * unit.reshape(40, 2, 32)[..., 0]).all()
    grid = np.concatenate([-R.GRID[::-1], R.GRID])
    best = np.abs(x[..., None] - grid * unit[..., None]).min(-1)
    np.testing.assert_allclose(np.abs(got - x), best, rtol=0, atol=1e-12 * np.abs(x).max())


def test_reference_plan_keeps_every_block_once():
    rng = np.random.default_rng(2)
    page, n = 4, 6
    old, q = rng.integers(0, 20, n), rng.integers(0, 9, n)
    fin = np.array([0, 1, 0, 0, 1, 0], bool)
    q[fin] = 0
    held = -(-old // page)
    order = rng.permutation(60)
    table = np.full((n, 9), -1)
    used = 0
    for r in range(n):
        table[r, :held[r]] = order[used:used + held[r]]
        used += held[r]
    free = np.full(60, -1)
    free[:60 - used] = order[used:]
    t, f, top, lens, cu, slots, pos, who = R.plan(page, old, q, fin, table, free, 60 - used)
    now = -(-np.array(lens) // page)
    kept = [t[r, :now[r]] for r in range(n)] + [f[:top]]
    assert sorted(np.concatenate(kept)) == list(range(60))
    assert len(set(slots)) == len(slots) == cu[-1] == q.sum()
    assert [lens[r] for r in who] >= [p + 1 for p in pos]
