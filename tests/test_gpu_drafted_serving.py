"""The example server that checks drafted trees: lengths, paths, blocks and cached rows."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_example_runs_and_accounts_for_every_block():
    from examples import drafted_serving

    r = drafted_serving.main(steps=25)
    assert r["tokens"] == r["lens"] and all(25 <= n <= 25 * 8 for n in r["lens"])
    assert r["free"] + r["held"] == r["blocks"]


def test_steps_keep_agreeing_paths_and_their_rows():
    import wohper_b200 as W
    from examples.drafted_serving import PARENTS, DraftServer

    ctx = W.Context(0)
    s = DraftServer(ctx, slots=3, layers=2, page=8, seed=3)
    s.learn()
    g = torch.Generator(device="cuda").manual_seed(4)
    texts = [[] for _ in range(s.slots)]
    roots = s.roots.tolist()
    for _ in range(9):
        random = torch.randint(0, 256, (s.slots, s.nodes), generator=g, device="cuda", dtype=torch.int32)
        drafts, targets, kept = s.step(random)
        d, t = drafts.view(s.slots, -1).tolist(), targets.view(s.slots, -1).tolist()
        path, counts = kept.path.view(s.slots, -1).tolist(), kept.counts.tolist()
        for r in range(s.slots):
            p = path[r][:counts[r]]
            assert p[0] == 0 and d[r][0] == roots[r] and path[r][counts[r]:] == [-1] * (s.nodes - counts[r])
            for a, b in zip(p, p[1:]):
                fits = [c for c in range(s.nodes) if PARENTS[c] == a and d[r][c] == t[r][a]]
                assert PARENTS[b] == a and fits[0] == b
            assert not [c for c in range(s.nodes) if PARENTS[c] == p[-1] and d[r][c] == t[r][p[-1]]]
            texts[r] += [d[r][j] for j in p]
            roots[r] = t[r][p[-1]]
        assert kept.next_tokens.tolist() == roots
    ctx.sync()
    lens = s.lens.tolist()
    assert lens == [len(x) for x in texts] and sum(lens) > 27  # some guesses were right
    held = sum(-(-n // s.page) for n in lens)
    used = [b for r, n in enumerate(lens) for b in s.table[r, :-(-n // s.page)].tolist()]
    assert int(s.top) + held == s.pool.blocks and len(set(used + s.free[:int(s.top)].tolist())) == s.pool.blocks
    # The first layer's rows depend on their tokens alone: row i is token i's, whatever tree it
    # came in.  4 bits hold a normed row to within about a tenth of its length; another
    # token's row would be at right angles to it.
    x = W.rms_norm(ctx, s.embed)
    want = W.rms_norm(ctx, W.gemm_fp8_e4m3_ue8m0(ctx, *s.wkv[0], x))
    for r, n in enumerate(lens):
        i = torch.arange(n, device="cuda")
        slots = s.table[r].long()[i // s.page] * s.page + i % s.page
        rows = W.kv_gather(ctx, s.caches[0], slots)[0].view(n, -1)
        near = torch.nn.functional.cosine_similarity(rows, want[torch.tensor(texts[r], device="cuda")], dim=1)
        assert float(near.min()) > 0.95
    ctx.close()
