"""CPU checks that sizes which a C int does not hold are refused by the drafted trees' calls,
the plan and the FP8 product (ctypes would hand on what is left of them: 2^32 + 5 as 5), and
that scratch sizes stay right up to there."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


class NoContext:
    """A context of GPU 0 without a handle."""
    device, handle = 0, None


@pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 5])
def test_sizes_past_32_bits_are_refused(n):
    import wohper_b200 as W

    def big(*shape, dtype=torch.int32):  # sizes without memory
        return torch.empty(shape, dtype=dtype, device="meta")

    ctx = NoContext()
    cache = W.PagedKvCache.empty(4, 16, 2, 128, True, device="cpu")
    one, two, table, top = big(1), big(2), big(1, 2), big(1)
    tree = W.KvTree(big(2, 1, dtype=torch.int64), two)
    q = torch.zeros(2, 4, 128)
    w, s = big(128, 128, dtype=torch.uint8), big(1, 1, dtype=torch.uint8)
    for what, call in (
            ("kv_lens", lambda: W.kv_tree(ctx, two, big(n + 1), big(n), 2)),
            ("parents", lambda: W.kv_tree(ctx, big(n), two, one, 2)),
            ("kv_lens", lambda: W.kv_tree_attention(ctx, cache, q, big(n + 1), big(n), big(n, 2), tree)),
            ("kv_lens", lambda: W.kv_attention(ctx, cache, q, big(n + 1), big(n), big(n, 2))),
            ("kv_lens", lambda: W.kv_accept(ctx, 16, two, two, two, big(n + 1), big(n), big(n, 2), two, top)),
            ("parents", lambda: W.kv_accept(ctx, 16, big(n), big(n), big(n), two, one, table, two, top)),
            ("free_blocks", lambda: W.kv_accept(ctx, 16, two, two, two, two, one, table, big(n), top)),
            ("kv_lens", lambda: W.kv_commit(ctx, cache, big(n), two, big(n + 1), big(n), big(n, 2))),
            ("path", lambda: W.kv_commit(ctx, cache, one, big(n), two, one, table)),
            ("kv_lens", lambda: W.kv_plan(ctx, 16, big(n), big(n), big(n, 2), two, top, 4)),
            ("free_blocks", lambda: W.kv_plan(ctx, 16, one, one, table, big(n), top, 4)),
            ("x", lambda: W.gemm_fp8_e4m3_ue8m0(ctx, w, s, big(n, 128, dtype=torch.bfloat16))),
            ("weight", lambda: W.gemm_fp8_e4m3_ue8m0(ctx, big(n, 16, dtype=torch.uint8), big(-(-n // 128), 1, dtype=torch.uint8),
                                                     big(2, 16, dtype=torch.bfloat16)))):
        with pytest.raises(W.WohperError) as e:
            call()
        assert e.value.kind == "InvalidShape" and f"{what}: {n} is past 32 bits" in str(e.value), e.value


def test_product_scratch_of_the_most_tokens_a_c_int_holds():
    import wohper_b200 as W

    size = W.lib().wh_fp8_gemm_scratch_bytes
    for tokens in ((1 << 30), (1 << 31) - 200, (1 << 31) - 1):
        for cols in (16, 8192, (1 << 31) - 16):
            tiles, ktiles = -(-tokens // 224), -(-cols // 128)
            assert tokens * cols + tiles * ktiles * 1024 <= size(cols, tokens) <= tokens * cols + 256 + 1024 * (tiles + 1) * ktiles
