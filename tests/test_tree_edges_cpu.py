"""Tree speculation without a GPU: refusals, rules and failures at the edges of the operators' arguments."""
import pytest
import torch

from carbon_b200.config import tiny_config
from carbon_b200.engine.engine import Engine
from carbon_b200.models.weights import WeightSource
from carbon_b200.ops import spec
from carbon_b200.ref.model import init_weights


def test_cache_rows_refuse_an_address_between_words():
    """The kernel moves rows in words of 4 bytes at least: a contiguous view that starts inside one is refused."""
    flat = torch.zeros(16 * 8 + 4, dtype=torch.uint8)
    base = flat.data_ptr()
    for off in range(4):
        view = flat[off:off + 128].view(16, 8)
        assert view.is_contiguous()
        if (base + off) % 4:
            with pytest.raises(ValueError, match="4-byte boundary"):
                spec.CacheRows([view])
            with pytest.raises(ValueError, match="4-byte boundary"):
                spec.CacheRows([torch.zeros(16, 4), view])
        else:
            spec.CacheRows([view])


@pytest.mark.parametrize("dtype", [torch.uint8, torch.bfloat16])
def test_rows_off_a_16_byte_boundary_are_refused(dtype):
    """What tree_mla asks of its cache before a launch (the row kernels read 16 bytes at a time)."""
    flat = torch.zeros(656 * 4 + 16, dtype=dtype)
    for off in range(0, 17):
        rows = flat[off:off + 656 * 4].view(4, 656)
        if rows.data_ptr() % 16:
            with pytest.raises(ValueError, match="16-byte boundary"):
                spec._aligned("tree_mla: kv", rows)
        else:
            spec._aligned("tree_mla: kv", rows)


# ----------------------------------------------------------------------------------------------------------------------
# the engine's step: failures
# ----------------------------------------------------------------------------------------------------------------------
def two_requests():
    cfg = tiny_config().replace(index_n_heads=0, index_topk=0)
    eng = Engine(cfg, "cpu", source=WeightSource(cfg, state=init_weights(cfg, seed=0)), num_pages=64, page_size=16)
    reqs = [eng.add_request([1, 2, 3]), eng.add_request([4, 5, 6, 7])]
    eng.prefill(reqs)
    return eng, reqs, [([5, 8, 9], [-1, 0, 0]), ([6, 3], [-1, 0])]


def state(reqs):
    return [(list(r.out), r.n_cached, r.seq_len) for r in reqs]


def test_a_wait_that_ran_out_fails_the_step():
    """The attention's status word (set here by hand, in the middle of the forward) ends the step with an error, and no
    request has grown."""
    eng, reqs, trees = two_requests()
    forward, before = eng.model.forward, state(reqs)

    def give_up(fb, cache):
        logits = forward(fb, cache)
        fb.tree.status.fill_(3)
        return logits

    eng.model.forward = give_up
    with pytest.raises(RuntimeError, match="status 3"):
        eng.verify_tree(reqs, trees)
    assert state(reqs) == before
    eng.model.forward = forward
    assert all(len(o) >= 1 for o in eng.verify_tree(reqs, trees))           # the next step starts with a clean word


def test_one_request_without_a_token_leaves_all_unchanged():
    """The second of two requests has no finite logits: the step raises, neither request has grown, and the step can be
    run again."""
    eng, reqs, trees = two_requests()
    forward, before = eng.model.forward, state(reqs)

    def spoil(fb, cache):
        logits = forward(fb, cache).clone()
        logits[3:] = float("nan")
        return logits

    eng.model.forward = spoil
    with pytest.raises(RuntimeError, match=f"request {reqs[1].rid}"):
        eng.verify_tree(reqs, trees)
    assert state(reqs) == before
    eng.model.forward = forward
    other, theirs, _ = two_requests()
    assert eng.verify_tree(reqs, trees) == other.verify_tree(theirs, trees)
    assert state(reqs) == state(theirs)


# ----------------------------------------------------------------------------------------------------------------------
# which calls expand their rows first
# ----------------------------------------------------------------------------------------------------------------------
def counts_of(requests, ctx, nodes, heads=128, page=64):
    """The counts of a plan whose requests share their pages."""
    from carbon_b200.ops._ext import available, ext

    if not available():
        pytest.skip("the extension is not built")
    table = list(range(-(-(ctx + nodes) // page)))
    code, _, counts, _ = ext().tree_plan([table] * requests, [ctx] * requests, [[-1] + [0] * (nodes - 1)] * requests, page,
                                         heads, 74)
    assert code == 0
    return counts


def test_expanded_rows_are_bounded():
    """A batch of fp8 requests expands its whole key tiles; one whose dense rows would pass the limit is fed instead, and
    so is what the rule never expands."""
    c = counts_of(32, 4096, 6)
    assert spec._stage_rows(c, True, 64, 576) == 32 * 4096 and spec._stage_rows(c, True, 64, 512) == 32 * 4096
    assert spec._stage_rows(c, False, 24, 576) == 32 * 4096
    assert spec._stage_rows(c, False, 64, 576) == 0                          # TMA takes them as they lie
    assert spec._stage_rows(counts_of(32, 4096, 1), True, 64, 576) == 0      # one row tile per key tile
    assert spec._stage_rows(counts_of(1, 700, 6), True, 64, 576) == 0        # few tiles
    for requests in (32, 64):                                                # 4.8 and 9.7 GB of dense rows
        assert spec._stage_rows(counts_of(requests, 131072, 6), True, 64, 576) == 0
    most = spec._STAGE_BYTES // (576 * 2 * 128)
    ok, over = counts_of(1, most * 128, 6), counts_of(1, (most + 1) * 128, 6)
    assert spec._stage_rows(ok, True, 64, 576) == most * 128 and spec._stage_rows(over, True, 64, 576) == 0


# ----------------------------------------------------------------------------------------------------------------------
# verification: tokens that are not in the vocabulary
# ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("probs", [False, True])
def test_tokens_outside_the_vocabulary_are_never_accepted(temperature, probs):
    """-1 and -5 would be the row's own last entries, 6 and 2^31 - 1 are past its end: none is accepted or changes what
    is left, and a sibling inside the vocabulary is tested as if alone."""
    logits = torch.tensor([[0.0, 1.0, 2.0, 3.0, 4.0, 9.0]]).repeat(7, 1)
    tokens = torch.tensor([0, -1, -5, 6, 2 ** 31 - 1, -2 ** 31, 5], dtype=torch.int32)
    for last in (5, -1):
        tokens[6] = last
        plan = spec.TreePlan([[0, 1]], [0], [[-1] + [0] * 6], 4, device="cpu")
        v = spec.tree_verify(logits, tokens, plan, torch.zeros(7), torch.ones(1, 6), torch.tensor([temperature]),
                             torch.full((7, 6), 1 / 6) if probs else None)
        assert v.n_accepted.tolist() == [int(last == 5)] and v.tokens[0, 0].item() == 5


def test_schedule_sends_a_one_tile_remainder_on():
    """27 and 10 key tiles over three pairs: at a share of 15 (13 tiles and 2 for an item's start and end) the first row
    tile is cut twice, and the single tile that is left goes to the pair with the least work like any other piece."""
    from carbon_b200.ops._ext import available, ext

    if not available():
        pytest.skip("the extension is not built")
    ctx = [27 * 128 - 1, 10 * 128 - 1]
    _, host, (used, items, *_), _ = ext().tree_plan([list(range(c // 64 + 1)) for c in ctx], ctx, [[-1], [-1]], 64, 16, 3)
    w, head = host.tolist(), (used + 4) // 4 * 4
    got = sorted(tuple(w[head + 8 * i + k] for k in (0, 2, 3)) for i in range(items))
    assert used == 3 and got == [(0, 0, 13), (0, 13, 13), (0, 26, 1), (1, 0, 10)]


class Long:
    """Drafts as many tokens as it is asked for: the known continuation, then zeros."""

    def __init__(self, full):
        self.full = full

    def propose(self, tokens, n):
        left = self.full[len(tokens):]
        return (left + [0] * n)[:n]

    def propose_tree(self, tokens, n):
        return self.propose(tokens, n), list(range(n))


@pytest.mark.parametrize("kw", [dict(tree=True), dict(temperature=1e-4), dict(tree=True, temperature=1e-4)])
def test_more_drafts_than_a_tree_holds(kw):
    """A drafter is asked for as many tokens as fit a tree (64 nodes with the pending one), however many the caller
    allows."""
    cfg = tiny_config().replace(index_n_heads=0, index_topk=0)
    w = init_weights(cfg, seed=0)
    make = lambda: Engine(cfg, "cpu", source=WeightSource(cfg, state=w), num_pages=64, page_size=16)
    prompt = [1, 2, 3, 4]
    ref = make().generate([prompt], 70)
    assert make().generate_speculative([prompt], 70, Long(prompt + ref[0]), n_draft=200, **kw) == ref
