"""A small server loop that checks trees of drafted tokens.

Every request brings a tree of eight tokens a step: the token that the last step ended
with, and guesses of what follows.  One step runs a toy model over all of them,

    plan     which blocks the nodes' rows go to                    (kv_plan)
    tree     each node's ancestors and position                    (kv_tree)
    project  queries and latent rows, FP8 weights                  (gemm_fp8_e4m3_ue8m0)
    append   the rows, quantised into their slots                  (kv_append)
    attend   each node over the cached rows and its ancestors      (kv_tree_attention)
    score    the model's own token after each node                 (lm_head_topk_score_batch)
    accept   the path that the model agrees with, blocks back      (kv_accept)
    commit   its rows to their places, all layers at once          (kv_commit)

with lengths, blocks and tokens on the GPU throughout, so the step is captured once in
a CUDA graph and replayed.  Weights are random; the guesses come from a table of what
the model says after each token alone, so many of them are right.

    python examples/drafted_serving.py
"""
from __future__ import annotations

import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

import wohper_b200 as W  # noqa: E402

# a guess along the table from nodes 0, 1, 3, 5 and a random one beside each
PARENTS = (-1, 0, 0, 1, 1, 3, 3, 5)
LIKELY = (1, 3, 5, 7)


class DraftServer:
    def __init__(self, ctx: W.Context, slots: int = 4, layers: int = 2, blocks: int = 160, page: int = 16,
                 heads: int = 8, head_dim: int = 512, hidden: int = 1024, vocab: int = 256,
                 most_blocks: int = 24, seed: int = 0, device: str = "cuda"):
        self.ctx, self.slots, self.page, self.heads, self.d, self.layers = ctx, slots, page, heads, head_dim, layers
        self.nodes = len(PARENTS)
        g = torch.Generator(device=device).manual_seed(seed)

        def fp8(rows, cols):
            w = torch.randn(rows, cols, generator=g, device=device) * 16
            scale = torch.full((-(-rows // 128), -(-cols // 128)), 127 - 9, dtype=torch.uint8, device=device)
            return w.to(torch.float8_e4m3fn).view(torch.uint8), scale

        self.embed = torch.randn(vocab, hidden, generator=g, device=device)
        self.lm_head = torch.randn(vocab, hidden, generator=g, device=device).bfloat16()
        self.wq = [fp8(heads * head_dim, hidden) for _ in range(layers)]
        self.wkv = [fp8(head_dim, hidden) for _ in range(layers)]
        self.wo = [fp8(hidden, heads * head_dim) for _ in range(layers)]
        # the layers lie inside a block: a cache for each, and one of all of them
        codes = torch.zeros(blocks, layers, page, head_dim // 2, dtype=torch.uint8, device=device)
        scales = torch.zeros(blocks, layers, page, head_dim // 32, dtype=torch.uint8, device=device)
        self.caches = [W.PagedKvCache(codes[:, i:i + 1], scales[:, i:i + 1]) for i in range(layers)]
        self.pool = W.PagedKvCache(codes, scales)
        i32 = dict(dtype=torch.int32, device=device)
        self.lens = torch.zeros(slots, **i32)
        self.table = torch.full((slots, most_blocks), -1, **i32)
        self.free = torch.arange(blocks, **i32)
        self.top = torch.tensor([blocks], **i32)
        self.roots = torch.arange(1, slots + 1, **i32)
        self.parents = torch.tensor(PARENTS * slots, **i32)
        self.q_lens = torch.full((slots,), self.nodes, **i32)
        self.follow = torch.zeros(vocab, **i32)

    def model(self, tokens, plan, tree):
        """The token that the model puts after each of `tokens` [n]."""
        ctx, n = self.ctx, tokens.numel()
        x = self.embed[tokens.long()]
        for cache, wq, wkv, wo in zip(self.caches, self.wq, self.wkv, self.wo):
            h = W.rms_norm(ctx, x)
            k = W.rms_norm(ctx, W.gemm_fp8_e4m3_ue8m0(ctx, *wkv, h)).view(n, 1, self.d)
            q = W.gemm_fp8_e4m3_ue8m0(ctx, *wq, h, out_dtype=torch.bfloat16).view(n, self.heads, self.d)
            W.kv_append(ctx, cache, plan.slots, k)
            o = W.kv_tree_attention(ctx, cache, q, plan.cu_q, plan.kv_lens, self.table, tree)
            x = x + 0.05 * W.gemm_fp8_e4m3_ue8m0(ctx, *wo, o.view(n, -1), out_dtype=torch.float32)
        return W.lm_head_topk_score_batch(ctx, self.lm_head, W.rms_norm(ctx, x), 1)[0].view(-1)

    def drafts(self, random):
        """The step's nodes: [slots, nodes], roots first."""
        t = random.clone()
        t[:, 0] = self.roots
        for node in LIKELY:
            t[:, node] = self.follow[t[:, PARENTS[node]].long()]
        return t

    def step(self, random):
        """One step; random int32 [slots, nodes]: the unlikely guesses.  Returns (drafts,
        targets, what was kept)."""
        ctx, tokens = self.ctx, self.slots * self.nodes
        drafts = self.drafts(random).view(-1)
        plan = W.kv_plan(ctx, self.page, self.lens, self.q_lens, self.table, self.free, self.top, tokens)
        tree = W.kv_tree(ctx, self.parents, plan.cu_q, plan.kv_lens, self.nodes)
        targets = self.model(drafts, plan, tree)
        kept = W.kv_accept(ctx, self.page, self.parents, drafts, targets, plan.cu_q, plan.kv_lens, self.table,
                           self.free, plan.free_top)
        W.kv_commit(ctx, self.pool, kept.counts, kept.path, plan.cu_q, plan.kv_lens, self.table)
        self.lens.copy_(kept.kv_lens)
        self.top.copy_(kept.free_top)
        self.roots.copy_(kept.next_tokens)
        return drafts, targets, kept

    def learn(self):
        """Fills the table of guesses: the model's token after each token alone."""
        n = self.slots
        one = torch.ones_like(self.q_lens)
        alone = torch.full((n,), -1, dtype=torch.int32, device=self.lens.device)
        vocab = self.follow.numel()
        for first in range(0, vocab, n):
            tokens = torch.arange(first, first + n, dtype=torch.int32, device=self.lens.device).clamp(max=vocab - 1)
            plan = W.kv_plan(self.ctx, self.page, self.lens, one, self.table, self.free, self.top, n)
            tree = W.kv_tree(self.ctx, alone, plan.cu_q, plan.kv_lens, 1)
            self.follow[first:first + n] = self.model(tokens, plan, tree)[:vocab - first]
        # (the rows were written into blocks that are still free: the stack's height was not taken over)

    def capture(self, random):
        """The step as a CUDA graph: (graph, what step returns); fill random, replay, read."""
        state = (self.lens, self.top, self.roots, self.table, self.free)
        before = [t.clone() for t in state]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # once as it is, to load the kernels; then the state as it was
            self.step(random)
            for t, b in zip(state, before):
                t.copy_(b)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = self.step(random)
        return graph, out


def main(steps: int = 20, seed: int = 0) -> dict:
    ctx = W.Context(0)
    s = DraftServer(ctx, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    s.learn()
    random = torch.zeros(s.slots, s.nodes, dtype=torch.int32, device="cuda")
    graph, (drafts, targets, kept) = s.capture(random)
    texts = [[] for _ in range(s.slots)]
    for _ in range(steps):
        random.copy_(torch.randint(0, s.follow.numel(), random.shape, generator=g, device="cuda"))
        graph.replay()
        path, counts, d = kept.path.view(s.slots, -1).tolist(), kept.counts.tolist(), drafts.view(s.slots, -1).tolist()
        for r in range(s.slots):
            texts[r] += [d[r][j] for j in path[r][:counts[r]]]
    ctx.sync()
    lens = s.lens.tolist()
    report = {"lens": lens, "tokens": [len(t) for t in texts], "a step": sum(lens) / (steps * s.slots),
              "free": int(s.top), "held": sum(-(-n // s.page) for n in lens), "blocks": s.pool.blocks}
    graph.reset()
    ctx.close()
    return report


if __name__ == "__main__":
    print(main())
