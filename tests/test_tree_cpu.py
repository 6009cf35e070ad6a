"""Tree speculation on the CPU oracle: plan layout and refusals, attention over branches, the verification walk (greedy
agreement, distribution of the emitted tokens, degenerate rows) and the commit of an accepted branch."""
import math

import pytest
import torch

from carbon_b200.ops import spec
from carbon_b200.ref import ops as R


def plan_of(parents, ctx, page=4, heads=2, masks=None, device="cpu"):
    tables, at = [], 1
    for p, c in zip(parents, ctx):
        k = max(1, -(-(c + len(p)) // page))
        tables.append(list(range(at, at + k))[::-1])
        at += k
    return spec.TreePlan(tables, ctx, parents, page, n_heads=heads, device=device, masks=masks), at * page


def test_plan_layout():
    plan, _ = plan_of([[-1, 0, 0, 1], [-1], []], [5, 0, 3])
    assert plan.cu.tolist() == [0, 4, 5, 5] and plan.T == 5 and plan.N == 4 and plan.B == 3
    assert plan.mask.tolist() == [1, 3, 5, 11, 1]
    assert plan.pos.tolist() == [5, 6, 6, 7, 0] and plan.req.tolist() == [0, 0, 0, 0, 1]
    # request 0 has pages [3, 2, 1]: positions 5..8 -> slots 9, 10, 11, 4
    assert plan.node_slots() == [9, 10, 11, 4, 16]


def test_plan_full_mask_bits():
    plan, _ = plan_of([[-1] + list(range(63))], [0])
    assert [x % (1 << 64) for x in plan.mask.tolist()] == [(1 << (i + 1)) - 1 for i in range(64)]


@pytest.mark.parametrize("kw,what", [
    (dict(parents=[[-1] + [0] * 64]), "at most 64"),
    (dict(parents=[[0, 0]]), "parent of node 0"),
    (dict(parents=[[-1, 1]]), "parent of node 1"),
    (dict(parents=[[-1, -1]]), "parent of node 1"),
    (dict(parents=[[-1, 0]], page_tables=[[1]], ctx=[3]), "pages for 4 positions"),
    (dict(parents=[[-1]], page_tables=[[-2, 1]]), "negative page"),
    (dict(parents=[[-1]], masks=[[2]]), "mask"),
    (dict(parents=[[-1]], masks=[[1, 1]]), "mask"),
    (dict(parents=[[-1], [-1]]), "one entry per request"),
    (dict(parents=[[-1]], ctx=[-1]), "pages for"),
    (dict(parents=[[-1]], page_size=0), "positive"),
])
def test_plan_refusals(kw, what):
    args = dict(page_tables=[[1, 2] * 20], ctx=[2], parents=[[-1]], page_size=4, device="cpu")
    args.update(kw)
    with pytest.raises(ValueError, match=what):
        spec.TreePlan(**args)


def test_attention_sees_context_and_branch():
    torch.manual_seed(0)
    par = [[-1, 0, 0, 1], [-1, 0]]
    plan, S = plan_of(par, [5, 0])
    q, kv = torch.randn(6, 2, 24), torch.randn(S, 24)
    out = spec.tree_mla(q, kv, plan, 0.3, 16)
    keys = kv[torch.tensor(plan.slots(0))]
    sel = keys[[0, 1, 2, 3, 4, 5, 6, 8]]                       # node 3: root, node 1, itself
    want = torch.softmax(q[3] @ sel.t() * 0.3, -1) @ sel[:, :16]
    torch.testing.assert_close(out[3], want)
    keys = kv[torch.tensor(plan.slots(1))]
    torch.testing.assert_close(out[4], keys[:1, :16].expand(2, 16))
    with pytest.raises(ValueError, match="nodes"):
        spec.tree_mla(q[:5], kv, plan, 0.3, 16)
    with pytest.raises(ValueError, match="slot"):
        spec.tree_mla(q, kv[:8], plan, 0.3, 16)


def test_attention_nothing_seen_is_zero():
    plan, S = plan_of([[-1, 0]], [0], masks=[[0, 2]])
    out = spec.tree_mla(torch.randn(2, 2, 24), torch.randn(S, 24), plan, 0.3, 16)
    assert bool((out[0] == 0).all()) and bool((out[1] != 0).any())


def verify(logits, tokens, parents, temperature, uniforms=None, noise=None, draft=None):
    n, V = logits.shape
    plan, _ = plan_of([parents], [0])
    u = torch.zeros(n) if uniforms is None else torch.tensor(uniforms)
    e = torch.ones(1, V) if noise is None else noise
    return spec.tree_verify(logits, torch.tensor(tokens, dtype=torch.int32), plan, u, e, torch.tensor([temperature]),
                            draft)


def test_verify_greedy_walks_the_agreeing_branch():
    V = 8
    best = [3, 5, 1, 2]
    logits = torch.zeros(4, V)
    for i, t in enumerate(best):
        logits[i, t] = 4.0
    # root's children: node 1 (token 6, wrong), node 2 (token 3, right); node 3 under node 2 carries token 1 (right)
    v = verify(logits, [0, 6, 3, 1], [-1, 0, 0, 2], 0.0)
    assert v.path.tolist() == [[0, 2, 3, -1]] and v.n_accepted.tolist() == [2]
    assert v.tokens.tolist() == [[3, 1, 2, -1]]
    want = 4.0 - math.log(math.exp(4.0) + 7)
    assert all(abs(x - want) < 1e-6 for x in v.logprobs[0, :3].tolist()) and v.logprobs[0, 3] == 0


def test_verify_ties_and_empty_rows():
    logits = torch.zeros(1, 6)
    assert verify(logits, [0], [-1], 0.0).tokens.tolist() == [[0]]
    assert verify(logits, [0], [-1], 1.0).tokens.tolist() == [[0]]          # equal noise: lowest index
    logits[0] = float("-inf")
    for t in (0.0, 1.0):
        v = verify(logits, [0], [-1], t)
        assert v.tokens.tolist() == [[-1]] and v.logprobs[0, 0] == float("-inf") and v.n_accepted.tolist() == [0]
    logits[0, 4] = 1.0                                                       # one token left by the mask
    assert verify(logits, [0], [-1], 0.7).tokens.tolist() == [[4]]


def test_verify_rejection_leaves_the_remainder():
    p = torch.tensor([0.5, 0.3, 0.2])
    q = torch.tensor([[0.9, 0.05, 0.05], [1 / 3] * 3])
    # token 0 accepted with probability 0.5 / 0.9; u above it rejects, the remainder is (0, 0.25, 0.15) / 0.4
    v = verify(p.log()[None].repeat(2, 1), [0, 0], [-1, 0], 1.0, uniforms=[0.0, 0.6], draft=q)
    assert v.n_accepted.tolist() == [0] and v.tokens[0, 0].item() == 1
    noise = torch.tensor([[1.0, 1.0, 0.5]])
    v = verify(p.log()[None].repeat(2, 1), [0, 0], [-1, 0], 1.0, uniforms=[0.0, 0.6], noise=noise, draft=q)
    assert v.tokens[0, 0].item() == 2                                        # 0.25 / 1 < 0.15 / 0.5
    v = verify(p.log()[None].repeat(2, 1), [0, 0], [-1, 0], 1.0, uniforms=[0.0, 0.5], draft=q)
    assert v.n_accepted.tolist() == [1] and v.tokens[0, 0].item() == 0


@pytest.mark.parametrize("with_draft", [False, True])
def test_verify_emits_the_target_distribution(with_draft):
    """The first emitted token of a three-child tree has the target's distribution, whatever was drafted: 20,000 draws
    against p, each frequency within 5 standard deviations (5 * sqrt(0.25 / 20000) = 0.018)."""
    torch.manual_seed(1)
    V, draws = 5, 20000
    p = torch.softmax(torch.randn(V), -1)
    q = torch.softmax(torch.randn(V), -1)
    kids = torch.multinomial(q, 3 * draws, replacement=True).view(draws, 3)
    u = torch.rand(draws, 4)
    e = torch.empty(draws, V).exponential_()
    hits = torch.zeros(V)
    lg = p.log()[None].expand(4, V)
    dp = q[None].expand(4, V) if with_draft else None
    for i in range(draws):
        kid = kids[i].tolist() if with_draft else [0, 3, 0]
        _, toks, _ = R.tree_verify(lg, [0] + kid, [-1, 0, 0, 0], u[i], e[i], 1.0, dp)
        hits[toks[0]] += 1
    assert ((hits / draws - p).abs() < 0.018).all(), (hits / draws, p)


def test_verify_shapes_refused():
    plan, _ = plan_of([[-1, 0]], [0])
    ok = dict(logits=torch.zeros(2, 6), tokens=torch.zeros(2, dtype=torch.int32), plan=plan, uniforms=torch.zeros(2),
              noise=torch.ones(1, 6), temperature=torch.zeros(1))
    spec.tree_verify(**ok)
    for name, bad in (("logits", torch.zeros(3, 6)), ("tokens", torch.zeros(1, dtype=torch.int32)),
                      ("uniforms", torch.zeros(3)), ("noise", torch.ones(1, 5)), ("temperature", torch.zeros(2)),
                      ("draft_probs", torch.zeros(2, 5))):
        with pytest.raises(ValueError, match=name):
            spec.tree_verify(**{**ok, name: bad})


def test_commit_moves_the_branch():
    plan, S = plan_of([[-1, 0, 0, 2, 2, 4], [-1, 0], [-1]], [6, 2, 0])
    a, b = torch.arange(S * 4.0).view(S, 4), torch.arange(S, dtype=torch.int32)
    rows = spec.CacheRows([a, None, b])
    at = plan.slots(0)[6:]
    before = b.clone()
    spec.tree_commit(rows, plan, torch.tensor([[0, 2, 4, 5, -1, -1], [0, -1, -1, -1, -1, -1], [0] + [-1] * 5]),
                     torch.tensor([3, 0, 0]))
    assert [b[at[k]].item() for k in range(1, 4)] == [before[at[k]].item() for k in (2, 4, 5)]
    assert (a[:, 0] == b * 4).all()
    keep = [s for s in range(S) if s not in at[1:4]]
    assert (b[keep] == before[keep]).all()
    with pytest.raises(ValueError, match="path"):
        spec.tree_commit(rows, plan, torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


def test_cache_rows_refusals():
    with pytest.raises(ValueError, match="no caches"):
        spec.CacheRows([None])
    with pytest.raises(ValueError, match="contiguous"):
        spec.CacheRows([torch.zeros(8, 4)[:, :2]])
    with pytest.raises(ValueError, match="4 bytes"):
        spec.CacheRows([torch.zeros(8, 3, dtype=torch.uint8)])


def test_native_plan_is_the_same():
    """The native builder's buffer behind the attention's work equals the Python lists; it refuses what they refuse."""
    from carbon_b200.ops._ext import available, ext

    if not available():
        pytest.skip("the extension is not built")
    parents = [[-1, 0, 0, 1, 3], [], [-1] + list(range(63)), [-1]]
    ctx, page = [5, 2, 130, 0], 7
    tables = [[3, 9], [4], list(range(20, 48)), [0, 77]]
    plan = spec.TreePlan(tables, ctx, parents, page, n_heads=16, device="cpu")
    code, host, counts, meta = ext().tree_plan(tables, ctx, parents, page, 16, 74)
    assert code == 0 and meta[1:] == [70, 64, 28, 77] and len(counts) == 7
    assert torch.equal(host[meta[0]:], plan._host)
    assert plan.node_slots() == [plan.slots(b)[ctx[b] + i] for b in range(4) for i in range(plan.n[b])]
    for bad in (dict(parents=[[-1, 1]] + parents[1:]), dict(ctx=[10, 2, 130, 0]), dict(ctx=[-1, 2, 130, 0]),
                dict(parents=[[-1] + [0] * 64] + parents[1:]), dict(tables=[[3, -9]] + tables[1:]), dict(ctx=[5]),
                dict(tables=[[3, 2 ** 31 // 7]] + tables[1:])):
        a = dict(tables=tables, ctx=ctx, parents=parents)
        a.update(bad)
        assert ext().tree_plan(a["tables"], a["ctx"], a["parents"], page, 16, 74)[0] == -1
        with pytest.raises(ValueError):
            spec.TreePlan(a["tables"], a["ctx"], a["parents"], page, n_heads=16, device="cpu")


@pytest.mark.parametrize("clusters,heads", [(74, 128), (74, 5), (1, 16), (7, 64)])
def test_schedule_covers_every_key_tile_once(clusters, heads):
    from carbon_b200.ops._ext import available, ext

    if not available():
        pytest.skip("the extension is not built")
    n = [1, 0, 6, 64, 17, 1]
    ctx = [0, 300, 127, 128, 9001, 4000]
    parents = [[-1] + [0] * (k - 1) if k else [] for k in n]
    tables = [list(range((c + k) // 64 + 1)) for c, k in zip(ctx, n)]
    _, host, (used, items, merges, parts, whole, work, most), meta = ext().tree_plan(tables, ctx, parents, 64, heads,
                                                                                     clusters)
    w = host[:meta[0]].tolist()
    first, head = w[:used + 1], (used + 4) // 4 * 4
    it = [w[head + 8 * i:head + 8 * i + 8] for i in range(items)]
    mg = [w[head + 8 * items + 6 * i:head + 8 * items + 6 * i + 6] for i in range(merges)]
    assert used <= clusters and first[0] == 0 and first[-1] == items and all(a < b for a, b in zip(first, first[1:]))
    cu = [sum(n[:b]) for b in range(len(n))]
    rows = {}
    for b, row, tile, tiles, part, c, c0, k in it:
        assert (c, c0, k) == (ctx[b], cu[b], n[b]) and tiles > 0
        rows.setdefault((b, row), []).append((tile, tiles, part))
    assert set(rows) == {(b, r) for b, k in enumerate(n) for r in range((k * heads + 127) // 128)}
    for (b, row), pieces in rows.items():
        at = 0
        for tile, tiles, _ in sorted(pieces):
            assert tile == at
            at += tiles
        assert at == (ctx[b] + n[b] + 127) // 128
        ids = sorted(p for _, _, p in pieces)
        if len(pieces) == 1:
            assert ids == [-1]
        else:
            assert [row, ids[0], len(ids), cu[b], n[b] * heads, 0] in mg and ids == list(range(ids[0], ids[0] + len(ids)))
    assert work == sum(x[3] for x in it) and parts == sum(m[2] for m in mg) and most == max([m[2] for m in mg] + [0])
    at = head + 8 * items + 6 * merges
    want = [(b, t) for b in range(len(n)) for t in range(ctx[b] // 128) if n[b]]
    assert whole == len(want) and [tuple(w[at + 2 * i:at + 2 * i + 2]) for i in range(whole)] == want
