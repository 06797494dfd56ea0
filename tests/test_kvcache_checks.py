"""CPU checks of what the paged 4-bit cache refuses before anything reaches the GPU."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


def refused(W, kind, why, fn, *a, **kw):
    with pytest.raises(W.WohperError) as e:
        fn(*a, **kw)
    assert e.value.kind == kind and why in str(e.value), e.value


def test_a_pool_whose_blocks_lie_on_one_another_is_refused():
    # a stride of 0 between several blocks is not a dense pool
    import wohper_b200 as W

    k = torch.zeros(1, 2, 5, 32, dtype=torch.uint8)
    s = torch.zeros(1, 2, 5, 2, dtype=torch.uint8)
    many = torch.zeros(3, 2, 5, 2, dtype=torch.uint8)
    W.PagedKvCache(k, s)
    W.PagedKvCache(k.expand(1, -1, -1, -1), s)
    refused(W, "InvalidShape", "stride", W.PagedKvCache, k.expand(3, -1, -1, -1), many)
    refused(W, "InvalidShape", "stride", W.PagedKvCache, torch.zeros(3, 2, 5, 32, dtype=torch.uint8),
            s.expand(3, -1, -1, -1))


@pytest.mark.parametrize("name", ["keys", "key_scales", "values", "value_scales"])
def test_a_pool_keeps_its_tensors(name):
    # the calls use the addresses of construction: another tensor is another cache
    import wohper_b200 as W

    c = W.PagedKvCache.empty(2, 4, 1, 64, True, device="cpu")
    old = getattr(c, name)
    with pytest.raises(AttributeError):
        setattr(c, name, torch.zeros_like(old))
    assert getattr(c, name) is old


class NoContext:
    """A context of GPU 0 without a handle: a call past its checks ends in "ctx is null"."""
    device, handle = 0, None


class NoStream:
    cuda_stream = 0


def test_tensors_that_are_not_on_the_contexts_gpu_are_refused():
    import wohper_b200 as W

    ctx, s = NoContext(), NoStream()
    cache = W.PagedKvCache.empty(4, 16, 2, 128, True, device="cpu")
    i32 = dict(dtype=torch.int32)
    lens, table = torch.ones(2, **i32), torch.zeros(2, 2, **i32)
    q, rows, slots = torch.zeros(2, 4, 128), torch.zeros(3, 2, 128), torch.arange(3)
    for stream in (None, s):
        refused(W, "InvalidPointer", "cuda:0", W.kv_plan, ctx, 16, lens, lens, table, torch.zeros(4, **i32),
                torch.zeros(1, **i32), 2, stream=stream)
        refused(W, "InvalidPointer", "cuda:0", W.kv_append, ctx, cache, slots, rows, rows, stream=stream)
        refused(W, "InvalidPointer", "cuda:0", W.kv_gather, ctx, cache, slots, stream=stream)
        refused(W, "InvalidPointer", "cuda:0", W.kv_attention, ctx, cache, q, None, lens, table, stream=stream)
