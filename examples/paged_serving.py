"""A small server loop on the paged 4-bit key/value cache.

Requests with prompts of different lengths arrive, get their prompt's rows in one
step and then one token a step, and leave; every step runs, for each layer,

    plan    which blocks the new tokens' rows go to           (kv_plan)
    norm    the new rows, as DeepSeek-V4 norms its latent rows  (rms_norm)
    append  the rows, quantised into their slots               (kv_append)
    attend  64 heads over each request's rows, the last `window` and the first
            `first` of them                                    (kv_attention)

with lengths, blocks and slots on the GPU throughout: the host never reads them
back, so a decode step is captured once in a CUDA graph and replayed.  Weights
and inputs are random; the point is the calls.

    python examples/paged_serving.py
"""
from __future__ import annotations

import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

import wohper_b200 as W  # noqa: E402


class PagedServer:
    """`slots` requests at a time over `layers` latent caches that share one block
    table (a block holds the same positions in every layer)."""

    def __init__(self, ctx: W.Context, slots: int = 8, layers: int = 2, blocks: int = 96,
                 page: int = 64, heads: int = 64, head_dim: int = 512, most_blocks: int = 16,
                 window: int = 128, first: int = 4, device: str = "cuda"):
        self.ctx, self.slots, self.page, self.heads, self.d = ctx, slots, page, heads, head_dim
        self.window, self.first = window, first
        # one pool; a layer's cache is a slice of it with a wider block stride
        codes = torch.zeros(blocks, layers, 1, page, head_dim // 2, dtype=torch.uint8, device=device)
        scales = torch.zeros(blocks, layers, 1, page, head_dim // 32, dtype=torch.uint8, device=device)
        self.caches = [W.PagedKvCache(codes[:, i], scales[:, i]) for i in range(layers)]
        i32 = dict(dtype=torch.int32, device=device)
        self.lens = torch.zeros(slots, **i32)
        self.table = torch.full((slots, most_blocks), -1, **i32)
        self.free = torch.arange(blocks, **i32)
        self.top = torch.tensor([blocks], **i32)
        self.gain = torch.ones(head_dim, dtype=torch.bfloat16, device=device)
        self.sink = torch.zeros(heads, device=device)

    def step(self, q_lens, rows, queries, finished=None):
        """One step.  q_lens int32 [slots]: new tokens of each request (0: none);
        rows[layer] f32 [tokens, head_dim]: their latent rows; queries[layer]
        [tokens, heads, head_dim]; finished uint8 [slots]: requests that leave.
        Returns the last layer's outputs [tokens, heads, head_dim]."""
        ctx, tokens = self.ctx, rows[0].shape[0]
        plan = W.kv_plan(ctx, self.page, self.lens, q_lens, self.table, self.free, self.top, tokens,
                         finished=finished)
        out = None
        for cache, x, q in zip(self.caches, rows, queries):
            k = W.rms_norm(ctx, x, self.gain).view(tokens, 1, self.d)
            W.kv_append(ctx, cache, plan.slots, k)
            out = W.kv_attention(ctx, cache, q, plan.cu_q, plan.kv_lens, self.table,
                                 window=self.window, first=self.first, sink=self.sink)
        self.lens.copy_(plan.kv_lens)
        self.top.copy_(plan.free_top)
        return out

    def capture(self, tokens: int):
        """The decode step of `tokens` tokens, one a request, as a CUDA graph: returns
        (graph, q_lens, rows, queries, out); fill the inputs, replay, read out."""
        dev = self.lens.device
        layers = len(self.caches)
        q_lens = torch.zeros(self.slots, dtype=torch.int32, device=dev)
        rows = [torch.zeros(tokens, self.d, device=dev) for _ in range(layers)]
        queries = [torch.zeros(tokens, self.heads, self.d, dtype=torch.bfloat16, device=dev)
                   for _ in range(layers)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # a step without tokens: loads the kernels, changes nothing
            self.step(q_lens, rows, queries)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = self.step(q_lens, rows, queries)
        return graph, q_lens, rows, queries, out


def main(steps: int = 12, seed: int = 0) -> dict:
    torch.manual_seed(seed)
    ctx = W.Context(0)
    s = PagedServer(ctx)
    dev = s.lens.device
    layers = len(s.caches)

    def inputs(n):
        return ([torch.randn(n, s.d, device=dev) for _ in range(layers)],
                [torch.randn(n, s.heads, s.d, device=dev).bfloat16() for _ in range(layers)])

    # prompts
    prompts = [70, 1, 200, 33, 128, 5, 64, 150]
    q_lens = torch.tensor(prompts, dtype=torch.int32, device=dev)
    s.step(q_lens, *inputs(sum(prompts)))
    ctx.sync()
    # decode, captured once
    graph, step_lens, rows, queries, out = s.capture(s.slots)
    step_lens.fill_(1)
    for _ in range(steps):
        r, q = inputs(s.slots)
        for a, b in zip(rows + queries, r + q):
            a.copy_(b)
        graph.replay()
    ctx.sync()
    lens = s.lens.cpu()
    # two requests leave, the others get another token
    gone = torch.zeros(s.slots, dtype=torch.uint8, device=dev)
    gone[1] = gone[4] = 1
    last = s.step((1 - gone).int(), *inputs(s.slots - 2), finished=gone)
    ctx.sync()
    held = -(-s.lens.cpu() // s.page)
    report = {"lens": lens.tolist(), "after": s.lens.cpu().tolist(), "free": int(s.top),
              "held": int(held.sum()), "blocks": s.caches[0].blocks,
              "finite": bool(torch.isfinite(out).all() and torch.isfinite(last).all())}
    graph.reset()
    ctx.close()
    return report


if __name__ == "__main__":
    print(main())
