"""Trees of drafted tokens over the paged 4-bit cache (``wh_kv_tree``,
``wh_kv_tree_attention``, ``wh_kv_accept``, ``wh_kv_commit``).

A step of a server that checks drafts, without a host synchronisation:

    plan = kv_plan(ctx, page, kv_lens, q_lens, block_table, free_blocks, free_top, tokens)
    tree = kv_tree(ctx, parents, plan.cu_q, plan.kv_lens, max_nodes)
    # per layer, with tree.positions for its rotary embedding
    kv_append(ctx, cache, plan.slots, k)
    out = kv_tree_attention(ctx, cache, q, plan.cu_q, plan.kv_lens, block_table, tree)
    # the model's own token after each node
    kept = kv_accept(ctx, page, parents, drafts, targets, plan.cu_q, plan.kv_lens, block_table,
                     free_blocks, plan.free_top)
    # per layer, or once for layers that lie inside a block
    kv_commit(ctx, cache, kept.counts, kept.path, plan.cu_q, plan.kv_lens, block_table)

Node j of a request (token cu_q[r] + j) has row base + j of the cache, base =
kv_lens[r] - its nodes.  The reference engine has no counterpart.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import Context, _check, lib
from .kvcache import (_INT_MAX, _INVALID_SHAPE, _UNSUPPORTED, PagedKvCache, _attend, _dense, _fail,
                      _handle, _int, _on, _on_gpu)

_I32 = torch.int32


@dataclass
class KvTree:
    """What kv_tree gives: masks int64 [tokens, words] (bit j: the token sees node j
    of its request) and positions int32 [tokens]."""
    masks: object
    positions: object


@dataclass
class KvAccept:
    """What kv_accept gives, int32: counts [requests] of kept nodes, path [tokens]
    (their indices from cu_q[r] on, then -1), next_tokens [requests], the new
    kv_lens [requests] and the stack's height free_top [1]."""
    counts: object
    path: object
    next_tokens: object
    kv_lens: object
    free_top: object


def _table(block_table, n: int, dev) -> int:
    if block_table.dim() != 2 or block_table.shape[0] != n:
        _fail(_INVALID_SHAPE, "block_table: [requests, max_blocks]")
    _int(block_table.shape[1], "block_table")
    _dense(block_table, _I32, block_table.numel(), dev, "block_table")
    return block_table.shape[1]


def kv_tree(ctx: Context, parents, cu_q, kv_lens, max_nodes: int, stream=None) -> KvTree:
    """Masks and positions of a step's drafted tokens (wh_kv_tree).  parents int32
    [tokens]: the parent's index inside the request, smaller than the node's own, or
    -1; cu_q and kv_lens as kv_plan gives them; max_nodes (at most 256): the most
    nodes of a request.  Bad parents and larger requests: ctx.sync() raises DeviceArg."""
    n, tokens, dev = kv_lens.numel(), parents.numel(), kv_lens.device
    _int(n, "kv_lens")
    _int(tokens, "parents")
    _on_gpu(ctx, dev, "kv_lens")
    _dense(kv_lens, _I32, n, dev, "kv_lens")
    _dense(cu_q, _I32, n + 1, dev, "cu_q")
    _dense(parents, _I32, tokens, dev, "parents")
    if not 1 <= max_nodes <= 256:
        _fail(_UNSUPPORTED, f"max_nodes {max_nodes}: 1 to 256")
    with _on(stream):
        masks = torch.empty((tokens, (max_nodes + 63) // 64), dtype=torch.int64, device=dev)
        positions = torch.empty(tokens, dtype=_I32, device=dev)
    _check(lib().wh_kv_tree(ctx.handle, n, tokens, max_nodes, parents.data_ptr(), cu_q.data_ptr(),
                            kv_lens.data_ptr(), masks.data_ptr(), positions.data_ptr(),
                            _handle(stream, dev)))
    return KvTree(masks, positions)


def kv_tree_attention(ctx: Context, cache: PagedKvCache, q, cu_q, kv_lens, block_table,
                      tree: KvTree, scale: Optional[float] = None, window: int = 0, first: int = 0,
                      sink=None, out=None, scratch=None, stream=None):
    """kv_attention where each query sees the cached rows before the step's (those
    inside the window that ends at its position, and the first ones) and the step's
    rows that its mask names (wh_kv_tree_attention).  A window has to be at least 64
    times the masks' words."""
    masks, words = tree.masks, tree.masks.shape[-1]
    if 0 < window < 64 * words:
        _fail(_UNSUPPORTED, f"window {window}: shorter than the tree's {64 * words}")
    return _attend(ctx, cache, q, cu_q, kv_lens, block_table, scale, window, first, sink, out,
                   scratch, stream, masks, tree.positions)


def kv_accept(ctx: Context, page: int, parents, drafts, targets, cu_q, kv_lens, block_table,
              free_blocks, free_top, stream=None) -> KvAccept:
    """The path of each request's tree that agrees with the model (wh_kv_accept):
    node 0, then on to the first child whose draft is its parent's target.  parents,
    drafts, targets int32 [tokens]; cu_q and kv_lens the step's (kv_plan).  Blocks
    past the new lengths go back on the stack free_blocks (height free_top [1]),
    which is updated in place; a stack that does not fit them changes nothing, keeps
    nothing, and ctx.sync() raises DeviceArg."""
    n, tokens, dev = kv_lens.numel(), parents.numel(), kv_lens.device
    _int(n, "kv_lens")
    _int(tokens, "parents")
    _int(free_blocks.numel(), "free_blocks")
    _on_gpu(ctx, dev, "kv_lens")
    _dense(kv_lens, _I32, n, dev, "kv_lens")
    _dense(cu_q, _I32, n + 1, dev, "cu_q")
    _dense(parents, _I32, tokens, dev, "parents")
    _dense(drafts, _I32, tokens, dev, "drafts")
    _dense(targets, _I32, tokens, dev, "targets")
    most = _table(block_table, n, dev)
    _dense(free_blocks, _I32, free_blocks.numel(), dev, "free_blocks")
    _dense(free_top, _I32, 1, dev, "free_top")
    if not 0 <= page <= _INT_MAX:
        _fail(_INVALID_SHAPE, f"page {page}")
    with _on(stream):  # counts | next | lens | top | path in one allocation
        ints = kv_lens.new_empty(3 * n + 1 + tokens)
    counts, nxt, lens, top, path = ints.split_with_sizes((n, n, n, 1, tokens))
    at = ints.data_ptr()
    _check(lib().wh_kv_accept(ctx.handle, n, page, most, tokens, parents.data_ptr(),
                              drafts.data_ptr(), targets.data_ptr(), cu_q.data_ptr(),
                              kv_lens.data_ptr(), block_table.data_ptr(), free_blocks.data_ptr(),
                              free_blocks.numel(), free_top.data_ptr(), at + 12 * n, at + 8 * n, at,
                              at + 12 * n + 4, at + 4 * n, _handle(stream, dev)))
    return KvAccept(counts, path, nxt, lens, top)


def kv_commit(ctx: Context, cache: PagedKvCache, counts, path, cu_q, kv_lens, block_table,
              stream=None) -> None:
    """Moves the rows of the kept nodes to their places (wh_kv_commit): row base +
    path[cu_q[r] + i] of request r becomes its row base + i, i < counts[r].  kv_lens
    is the step's, before kv_accept.  A pool [blocks, layers, kv_heads, page, ..]
    may be given as one cache of layers * kv_heads heads."""
    n, dev = kv_lens.numel(), cache.keys.device
    _int(n, "kv_lens")
    _int(path.numel(), "path")
    _on_gpu(ctx, dev, "cache")
    _dense(kv_lens, _I32, n, dev, "kv_lens")
    _dense(counts, _I32, n, dev, "counts")
    _dense(cu_q, _I32, n + 1, dev, "cu_q")
    _dense(path, _I32, path.numel(), dev, "path")
    _check(lib().wh_kv_commit(ctx.handle, cache._ref, n, path.numel(), counts.data_ptr(),
                              path.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(),
                              block_table.data_ptr(), _table(block_table, n, dev),
                              _handle(stream, dev)))
