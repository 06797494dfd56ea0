"""CPU checks of what the drafted trees' calls and the FP8 product refuse before anything
reaches the GPU, and of the plain forms that the GPU tests use."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests import tree_reference as T

torch = pytest.importorskip("torch")


class NoContext:
    """A context of GPU 0 without a handle."""
    device, handle = 0, None


def refused(W, kind, why, fn, *a, **kw):
    with pytest.raises(W.WohperError) as e:
        fn(*a, **kw)
    assert e.value.kind == kind and why in str(e.value), e.value


def test_tensors_that_are_not_on_the_contexts_gpu_are_refused():
    import wohper_b200 as W

    ctx = NoContext()
    cache = W.PagedKvCache.empty(4, 16, 2, 128, True, device="cpu")
    i32 = dict(dtype=torch.int32)
    lens, cu, table, nodes = torch.ones(2, **i32), torch.zeros(3, **i32), torch.zeros(2, 2, **i32), torch.zeros(5, **i32)
    tree = W.KvTree(torch.zeros(5, 1, dtype=torch.int64), nodes)
    at = "cuda:0"
    refused(W, "InvalidPointer", at, W.kv_tree, ctx, nodes, cu, lens, 5)
    refused(W, "InvalidPointer", at, W.kv_tree_attention, ctx, cache, torch.zeros(5, 4, 128), cu, lens, table, tree)
    refused(W, "InvalidPointer", at, W.kv_accept, ctx, 16, nodes, nodes, nodes, cu, lens, table, torch.zeros(4, **i32), lens[:1])
    refused(W, "InvalidPointer", at, W.kv_commit, ctx, cache, lens, nodes, cu, lens, table)
    w = torch.zeros(128, 128, dtype=torch.uint8)
    refused(W, "InvalidPointer", at, W.gemm_fp8_e4m3_ue8m0, ctx, w, w[:1, :1], torch.zeros(2, 128))
    refused(W, "Unsupported", "shorter than the tree", W.kv_tree_attention, ctx, cache, torch.zeros(5, 4, 128), cu, lens, table, tree,
            window=63)


def test_c_calls_without_a_context():
    import wohper_b200 as W

    L = W.lib()
    n = None
    assert L.wh_kv_tree(n, 1, 1, 1, n, n, n, n, n, n) == 9
    assert L.wh_kv_tree_attention(n, n, n, 0, 1, 1, 0, 0, 1, n, n, n, 1, n, 1, n, 1.0, 0, 0, n, n, 0, 0, n, 0, n) == 9
    assert L.wh_kv_accept(n, 1, 1, 1, 1, n, n, n, n, n, n, n, 1, n, n, n, n, n, n, n) == 9
    assert L.wh_kv_commit(n, n, 1, 1, n, n, n, n, n, 1, n) == 9
    assert L.wh_fp8_gemm(n, n, n, 1, 16, 1, 1, n, 0, 1, 16, n, 0, 1, 64, n, 0, n) == 9


def test_gemm_scratch_holds_codes_and_scale_tiles():
    import wohper_b200 as W

    size = W.lib().wh_fp8_gemm_scratch_bytes
    # few tokens are quantised by the product itself
    assert size(0, 9) == size(16, 0) == size(-1, -1) == size(4096, 1) == size(4096, 2) == 0
    for cols, tokens in ((16, 5), (1360, 257), (8192, 100000)):
        ktiles = -(-cols // 128)
        for tile, block in ((16, 512), (32, 512), (64, 512), (128, 512), (224, 1024)):
            if tile >= 128 or tokens <= tile:
                assert size(cols, tokens) >= tokens * cols + -(-tokens // tile) * ktiles * block
    assert size(32768, 1 << 20) > 1 << 35  # past 32 bits


def test_the_plain_tree():
    parents = np.array([-1, 0, 0, 2, 3, -1, 0, 1], np.int32)
    masks, pos = T.tree(parents, [0, 5, 8], [15, 4], 8, 1)
    assert masks[:, 0].tolist() == [1, 3, 5, 13, 29, 1, 3, 7]
    assert pos.tolist() == [10, 11, 11, 12, 13, 1, 2, 3]
    counts, path, nxt, after, free, top = T.accept(4, parents, [9, 1, 1, 4, 2, 9, 7, 3], [1, 5, 4, 2, 6, 8, 7, 0], [0, 5, 8], [15, 4],
                                                   np.arange(8).reshape(2, 4), np.full(3, -1), 1)
    # request 0: node 1 fits before node 2 and ends there; request 1: no child's draft is 8
    assert (counts, nxt, after, top) == ([2, 1], [5, 8], [12, 2], 2)
    assert path.tolist() == [0, 1, -1, -1, -1, 0, -1, -1] and free.tolist() == [-1, 3, -1]


def test_every_call_is_bound_with_its_argument_count():
    import re
    from pathlib import Path

    import wohper_b200 as W

    header = (Path(__file__).resolve().parents[1] / "include" / "wohper_b200.h").read_text()
    for name in ("wh_kv_tree", "wh_kv_tree_attention", "wh_kv_accept", "wh_kv_commit", "wh_fp8_gemm", "wh_fp8_gemm_scratch_bytes"):
        args = re.search(rf"\b{name}\(([^;]*?)\);", header, re.S).group(1).split(",")
        kinds = getattr(W.lib(), name).argtypes
        assert len(kinds) == len(args), name
        for a, k in zip(args, kinds):
            want = C.c_void_p if "*" in a or "wh_stream_t" in a else C.c_longlong if "long long" in a else \
                C.c_size_t if "size_t" in a else C.c_float if "float" in a else C.c_int
            assert k is want, (name, a, k)
