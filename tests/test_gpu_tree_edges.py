"""Tree-speculation kernels at the edges of their arguments' ranges, against the definitions in 64 bits."""
import pytest
import torch

from test_gpu_tree import (DEV, SCALE, check_verify, close, engine_cfg, exact, inputs, make_plan, rows_of, tree,
                           verify_inputs)
from carbon_b200.ops import spec

pytestmark = pytest.mark.gpu
LAST = 1 - 2.0 ** -24                                                       # the largest fp32 below 1


# ----------------------------------------------------------------------------------------------------------------------
# verification: what is left after a rejection
# ----------------------------------------------------------------------------------------------------------------------
def drafted_rows(B, kids, V, seed, dtype, filler):
    """B requests, a root with ``kids`` children whose tokens are spread over the vocabulary; every other token of the
    root's row has the logit ``filler``."""
    g = torch.Generator().manual_seed(seed)
    n = kids + 1
    logits = torch.randn(B, n, V, generator=g)
    logits[:, 0] = filler
    tok = torch.zeros(B, n, dtype=torch.int32)
    for b in range(B):
        tok[b, 1:] = torch.randperm(V, generator=g)[:kids].int()
        logits[b, 0, tok[b, 1:].long()] = torch.rand(kids, generator=g) * 4 - 2
    kw = dict(logits=logits.view(B * n, V).to(dtype), tokens=tok.view(-1), uniforms=torch.zeros(B, n),
              noise=torch.empty(B, V).exponential_(generator=g), temperature=torch.full((B,), 0.8), draft_probs=None)
    return [[-1] + [0] * kids] * B, kw


@pytest.mark.parametrize("V", [3, 500, 9000, 70001])
@pytest.mark.parametrize("kids", [2, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tree_verify_drafts_hold_all_the_mass(V, kids, dtype):
    """Only the drafted tokens are allowed: after the others are rejected the last one has probability 1 and is
    accepted at every number below 1."""
    parents, kw = drafted_rows(40, kids, V, V + kids, dtype, float("-inf"))
    kw["uniforms"][:, 1:] = LAST
    kw["uniforms"] = kw["uniforms"].view(-1)
    v = check_verify(parents, kw)
    assert bool((v.n_accepted == 1).all()) and bool((v.path[:, 1] == kids).all())


def test_tree_verify_two_allowed_tokens():
    lg = torch.full((3, 500), float("-inf"))
    lg[0, 0], lg[0, 1] = -1.4074705, -2.530843
    lg[1:, 7] = 0
    for V in (2, 500):
        lv = lg[:, :V].clone()
        lv[1:, 0] = 0
        v = check_verify([[-1, 0, 0]], dict(logits=lv, tokens=torch.tensor([0, 0, 1], dtype=torch.int32),
                                            uniforms=torch.tensor([0, 0.9, LAST]), noise=torch.ones(1, V),
                                            temperature=torch.tensor([0.8]), draft_probs=None))
        assert v.path[0, :2].tolist() == [0, 2]


@pytest.mark.parametrize("V", [500, 70001])
def test_tree_verify_remainder_of_a_peaked_row(V):
    """The first child holds all but 1e-3 to 1e-5 of the mass; the second is tested against what is left.  Its share
    x / (sum of the rest) has the rounding of exponents up to 20 (20 * 2^-22 = 5e-6) and of the sum (1e-6): numbers
    2e-5 below and above the 64-bit share are accepted and rejected."""
    B = 40
    for sign, taken in ((-1, 1), (1, 0)):
        parents, kw = drafted_rows(B, 2, V, V, torch.float32, -8.0)
        rows = kw["logits"].view(B, 3, V)
        g = torch.Generator().manual_seed(V)
        for b in range(B):
            a, x = kw["tokens"][3 * b + 1:3 * b + 3].long().tolist()
            rest = torch.rand((), generator=g).item() * 3
            rows[b, 0, x] = torch.log(torch.tensor(float(V))) * 0.8 - 8.0 + rest
            rows[b, 0, a] = rows[b, 0].div(0.8).logsumexp(0) * 0.8 + 0.8 * (7 + 4 * torch.rand((), generator=g).item())
            p = (rows[b, 0].double() / 0.8).softmax(0)
            p[a] = 0
            kw["uniforms"][b, 1] = LAST
            kw["uniforms"][b, 2] = (p[x] / p.sum()).item() * (1 + sign * 2e-5)
        kw["uniforms"] = kw["uniforms"].view(-1)
        v = check_verify(parents, kw)
        assert bool((v.n_accepted == taken).all())


def test_tree_verify_wide_roots_and_repeated_tokens():
    """63 children of one node, some with the same token, with certain proposals: drawn numbers and numbers near 1."""
    g = torch.Generator().manual_seed(11)
    for V, top in ((40, 1.0), (3000, LAST)):
        parents, kw = drafted_rows(12, 40 if V == 40 else 63, V, V, torch.float32, -3.0)
        n = len(parents[0])
        tok = kw["tokens"].view(12, n)
        tok[:, 5::3] = tok[:, 4:5]                                          # repeats of node 4's token
        kw["uniforms"] = (torch.rand(12 * n, generator=g) * top).clamp(max=LAST)
        check_verify(parents, kw)


def test_tree_verify_a_first_child_whose_own_drafts_hold_the_mass():
    """The same two levels down: the accepted first child's row, whose sums may come with its parent's."""
    B = 32
    for V in (60, 900, 30000):
        g = torch.Generator().manual_seed(V)
        parents = [[-1, 0, 1, 1]] * B
        logits = torch.full((B, 4, V), float("-inf"))
        tok = torch.zeros(B, 4, dtype=torch.int32)
        for b in range(B):
            tok[b, 1:] = torch.randperm(V, generator=g)[:3].int()
            logits[b, 0, tok[b, 1].long()] = 1.0
            logits[b, 1, tok[b, 2:].long()] = torch.rand(2, generator=g) * 4 - 2
            logits[b, 2:, 1] = 0.5
        u = torch.tensor([0.0, LAST, LAST, LAST]).repeat(B)
        v = check_verify(parents, dict(logits=logits.view(-1, V), tokens=tok.view(-1), uniforms=u,
                                       noise=torch.empty(B, V).exponential_(generator=g),
                                       temperature=torch.full((B,), 0.8), draft_probs=None))
        assert bool((v.path[:, :3] == torch.tensor([0, 1, 3])).all())


@pytest.mark.parametrize("heat", [float("inf"), 3e38, 1e-30, 1e-40])
@pytest.mark.parametrize("probs", [False, True])
def test_tree_verify_extreme_temperatures(heat, probs):
    """Every positive temperature has a distribution: uniform where it is infinite, the maximum as it goes to zero
    (1e-40 is subnormal in fp32)."""
    parents = [tree(5, i) for i in range(6)]
    check_verify(parents, verify_inputs(parents, 3000, 21, probs, temps=(heat,)))


# ----------------------------------------------------------------------------------------------------------------------
# attention: where rows begin
# ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("f8,page", [(False, 64), (False, 24), (True, 64)])
def test_tree_mla_rows_off_a_16_byte_boundary(f8, page):
    """A cache that starts off a 16-byte boundary is refused on the host; queries that do are copied."""
    plan, S = make_plan([tree(6, 0)], [300], page, 16)
    q, kv, _ = inputs(plan, S, 16, 576, f8, seed=3)
    want = spec.tree_mla(q, kv, plan, SCALE)
    for off in (1, 4) if f8 else (1, 2, 4):
        flat = torch.empty(kv.numel() + 16, dtype=kv.dtype, device=DEV)
        moved = flat[off:off + kv.numel()].view(kv.shape)
        with pytest.raises(ValueError, match="16-byte boundary"):
            spec.tree_mla(q, moved, plan, SCALE)
        flat = torch.empty(q.numel() + 16, dtype=q.dtype, device=DEV)
        moved = flat[off:off + q.numel()].view(q.shape)
        moved.copy_(q)
        assert torch.equal(spec.tree_mla(moved, kv, plan, SCALE), want)


# ----------------------------------------------------------------------------------------------------------------------
# attention over rows that are expanded to dense tiles first
# ----------------------------------------------------------------------------------------------------------------------
STAGED = [
    # contexts (nodes 6, the fourth request has none), heads, width, fp8, page, sink
    ([1501, 1280, 127, 900, 1999, 128, 1407, 1153, 640, 1663, 1282, 1700], 128, 576, True, 64, False),
    ([1501, 1280, 127, 900, 1999, 128, 1407, 1153, 640, 1663, 1282, 1700], 128, 512, True, 64, True),
    ([1501, 1280, 127, 900, 1999, 128, 1407, 1153, 640, 1663, 1282, 1700], 128, 576, False, 24, True),
    ([1501, 1280, 127, 900, 1999, 128, 1407, 1153, 640, 1663, 1282, 1700], 128, 512, False, 5, False),
    ([1501, 1280, 127, 900, 1999, 128, 1407, 1153, 640, 1663, 1282, 1700], 128, 576, True, 7, True),
    ([9000], 128, 576, True, 64, False),
]


def staged_plan(ctx, H, page, nodes=6):
    n = [0 if b == 3 else nodes for b in range(len(ctx))]
    return make_plan([tree(k, i) if k else [] for i, k in enumerate(n)], ctx, page, H)


@pytest.mark.parametrize("ctx,H,D,f8,page,sink", STAGED)
def test_tree_mla_expanded_rows(ctx, H, D, f8, page, sink):
    plan, S = staged_plan(ctx, H, page, 33 if len(ctx) == 1 else 6)
    assert spec._stage_rows(plan._counts, f8, page, D) == 128 * sum(c // 128 for b, c in enumerate(ctx) if b != 3)
    q, kv, sk = inputs(plan, S, H, D, f8, seed=D + page, sink=sink)
    close(spec.tree_mla(q, kv, plan, SCALE, sink=sk), exact(q, kv, plan, SCALE, sk))


@pytest.mark.parametrize("D,page,f8", [(576, 64, True), (512, 64, True), (576, 24, False), (512, 5, False)])
def test_tree_mla_expanded_rows_garbage_outside_the_mask(D, page, f8):
    """Unwritten rows and nodes of other branches that hold NaN and infinities do not reach a node that does not see
    them."""
    ctx = [1501, 1280, 127, 900, 1999, 128, 1407, 1153, 640, 1663, 1282, 1700]
    masks = [[(1 << i) | 1 for i in range(6)] if b != 3 else [] for b in range(12)]     # the root and itself
    plan, S = make_plan([tree(6, b) if b != 3 else [] for b in range(12)], ctx, page, 128, masks=masks)
    assert spec._stage_rows(plan._counts, f8, page, D)
    q, kv, _ = inputs(plan, S, 128, D, f8, seed=31)
    want = exact(q, kv, plan, SCALE)
    live = torch.zeros(S, dtype=torch.bool, device=DEV)
    rows, at = [], 0
    for b in range(12):
        slots = torch.tensor(plan.slots(b), device=DEV, dtype=torch.long)
        live[slots] = True
        if b != 3:
            live[slots[ctx[b] + 4]] = False                                 # node 4 of every tree: seen by itself alone
            rows += [at + i for i in (0, 1, 2, 3, 5)]
            at += 6
    kv[~live] = 0x7F if f8 else float("nan")
    if not f8:
        kv[~live, ::2] = float("inf")
    got = spec.tree_mla(q, kv, plan, SCALE)
    close(got[rows], want[rows])
    assert bool(torch.isnan(got[4::6]).all())


# ----------------------------------------------------------------------------------------------------------------------
# the engine's step, row by row
# ----------------------------------------------------------------------------------------------------------------------
def dense_engine(kind, **kw):
    """A model without routed experts: no router choice can flip between two ways of computing a row."""
    from carbon_b200.engine.engine import Engine
    from carbon_b200.models.weights import WeightSource
    from carbon_b200.ref.model import init_weights

    cfg = engine_cfg(kind)
    cfg = cfg.replace(n_dense_layers=cfg.n_layers)
    src = WeightSource(cfg, state=init_weights(cfg, seed=0))
    return cfg, lambda: Engine(cfg, device="cuda", source=src, num_pages=96, page_size=64, **kw)


@pytest.mark.parametrize("kind", ["dense", "dense_fp8", "latent"])
def test_engine_attention_of_every_node_and_layer(kind, monkeypatch):
    """The attention of every layer of a tree step, node by node, against the definition in 64 bits over the request's
    pages: the context's rows and those of the node's own branch, found from the trees and the page tables alone."""
    from carbon_b200.models import deepseek

    cfg, make = dense_engine(kind)
    g = torch.Generator().manual_seed(1)
    ps = [torch.randint(0, cfg.vocab_size, (k,), generator=g).tolist() for k in (70, 131, 300)]
    trees = [([5, 6, 7, 8], [-1, 0, 0, 1]), ([9], [-1]), ([1, 2, 3, 4, 5, 6], [-1, 0, 1, 1, 2, 0])]
    eng = make()
    reqs = [eng.add_request(p) for p in ps]
    eng.prefill(reqs)
    calls, plain = [], spec.tree_mla

    def record(q, kv, plan, scale, r, sink=None):
        out = plain(q, kv, plan, scale, r, sink=sink)
        calls.append((q.double(), kv.clone(), scale, sink, out.clone()))
        return out

    monkeypatch.setattr(deepseek.S, "tree_mla", record)
    eng.verify_tree(reqs, trees)
    assert len(calls) == cfg.n_layers
    for q, kv, scale, sink, out in calls:
        t = 0
        for req, p, (toks, par) in zip(reqs, ps, trees):
            for i in range(len(toks)):
                branch, k = [], i
                while k >= 0:
                    branch.insert(0, k)
                    k = par[k]
                at = list(range(len(p))) + [len(p) + k for k in branch]
                slots = torch.tensor([req.pages[x // 64] * 64 + x % 64 for x in at], device=DEV)
                keys = rows_of(kv[slots], q.shape[2]).double()
                s = q[t] @ keys.t() * scale
                if sink is not None:
                    s = torch.cat([s, sink.double()[:, None]], 1)
                close(out[t], torch.softmax(s, 1)[:, :len(at)] @ keys[:, :512])
                t += 1
        assert t == q.shape[0]


@pytest.mark.parametrize("kind", ["dense", "dense_fp8", "latent", "dsa"])
def test_engine_every_node_is_nearest_its_own_branch(kind):
    """The logits of every node of a tree step against all the nodes' branches run as decode rows: its own is the
    nearest.  (How far is not asserted: roundings that differ move a row by some percent through the fp8 products.)"""
    cfg, make = dense_engine(kind)
    g = torch.Generator().manual_seed(1)
    ps = [torch.randint(0, cfg.vocab_size, (k,), generator=g).tolist() for k in (70, 131, 300)]
    trees = [([5, 6, 7, 8], [-1, 0, 0, 1]), ([9], [-1]), ([1, 2, 3, 4, 5, 6], [-1, 0, 1, 1, 2, 0])]
    eng, rows = make(), []
    for p, (toks, par) in zip(ps, trees):
        for i in range(len(toks)):
            branch, k = [], i
            while k >= 0:
                branch.insert(0, toks[k])
                k = par[k]
            r = eng.add_request(p)
            eng.prefill([r])
            for t in branch:
                lg = eng.decode([r], [t])
            rows.append(lg[0].float())
            eng.release(r)
    reqs = [eng.add_request(p) for p in ps]
    eng.prefill(reqs)
    seen = {}
    forward = eng.model.forward

    def keep(fb, cache):
        seen["logits"] = forward(fb, cache).clone()
        return seen["logits"]

    eng.model.forward = keep
    eng.verify_tree(reqs, trees)
    want = torch.stack(rows)
    assert torch.cdist(seen["logits"].float(), want).argmin(1).tolist() == list(range(len(want)))


@pytest.mark.parametrize("kind", ["dense", "dense_fp8", "latent", "dsa"])
def test_engine_greedy_trees_follow_the_target(kind):
    """Greedy trees from prompt lookup and from the target itself: replayed token by token through plain decoding, every
    emitted token is the target's best but for rounding.  The GPU model's logits are within 12 % of the oracle's norm,
    0.12 rms a logit; three standard deviations of the difference of two are 0.12 * sqrt(2) * 3 = 0.5 rms."""
    from carbon_b200.engine.spec import ModelDrafter, NgramDrafter

    cfg, make = dense_engine(kind)
    g = torch.Generator().manual_seed(2)
    base = torch.randint(0, cfg.vocab_size, (20,), generator=g).tolist()
    ps = [base * 3, torch.randint(0, cfg.vocab_size, (280,), generator=g).tolist()]
    for drafter in (NgramDrafter(), ModelDrafter(make())):
        outs = make().generate_speculative(ps, 10, drafter, n_draft=6, tree=True)
        eng = make()
        reqs = [eng.add_request(p) for p in ps]
        logits = eng.prefill(reqs).float()
        for i in range(10):
            tok = [o[i] for o in outs]
            short = logits.amax(-1) - logits[torch.arange(2), tok]
            assert bool((short <= 0.5 * logits.pow(2).mean(-1).sqrt()).all()), (i, short)
            if i < 9:
                logits = eng.decode(reqs, tok).float()
