"""Tree speculation through the engine (CPU oracle): greedy trees give exactly the tokens of plain decoding, whatever was
drafted and whichever branch is accepted, in every attention layout; sampling is reproducible and needs one rank."""
import pytest
import torch

from carbon_b200.config import tiny_config, tiny_v4_config
from carbon_b200.engine.engine import Engine
from carbon_b200.engine.spec import ModelDrafter, NgramDrafter
from carbon_b200.models.weights import WeightSource
from carbon_b200.ref.model import init_weights

LAYOUTS = {
    "mla": tiny_config(),                                                    # DSA over the path's key list
    "mla_dense": tiny_config().replace(index_n_heads=0, index_topk=0),       # tree attention in every layer
    "mla_short": tiny_config().replace(index_topk=512),                      # fewer keys than top-k: tree attention
    "mla_fp8": tiny_config().replace(index_n_heads=0, index_topk=0, kv_fp8=True, attn_sink=True),
    "v4": tiny_v4_config(),                                                  # latent MQA, window, shared selections
    "latent_dense": tiny_v4_config().replace(swa_window=0, index_n_heads=0, index_topk=0, index_sources=()),
    "engram": tiny_config().replace(engram_layers=(1,), engram_heads=2, engram_dim=32, engram_rows=64),
}


def make(cfg, w, **kw):
    return Engine(cfg, "cpu", source=WeightSource(cfg, state=w), num_pages=64, page_size=16, **kw)


class Forked:
    """Drafts trees from a known continuation: a wrong first child at every level, the right token second, and a leaf
    under the wrong one."""

    def __init__(self, sequences):
        self.sequences = sequences

    def propose_tree(self, tokens, n):
        full = next(s for s in self.sequences if s[:len(tokens)] == list(tokens))
        out, parents, at = [], [], 0
        for t in full[len(tokens):]:
            if len(out) + 3 > n:
                break
            out += [(t + 1) % 997, t, (t + 2) % 997]
            parents += [at, at, len(out) - 2]
            at = len(out) - 1
        return out, parents


def prompts(vocab):
    g = torch.Generator().manual_seed(3)
    base = torch.randint(0, vocab, (20,), generator=g).tolist()
    return [base * 3, torch.randint(0, vocab, (37,), generator=g).tolist()]


@pytest.mark.parametrize("name", list(LAYOUTS))
def test_greedy_trees_match_greedy(name):
    cfg = LAYOUTS[name]
    w = init_weights(cfg, seed=0)
    ps = prompts(cfg.vocab_size)
    ref = make(cfg, w).generate(ps, 14)
    eng = make(cfg, w)
    out = eng.generate_speculative(ps, 14, Forked([p + o for p, o in zip(ps, ref)]), n_draft=9, tree=True)
    assert out == ref
    assert eng.stats["verify_steps"] <= 6                    # three right tokens and the next one per step
    assert make(cfg, w).generate_speculative(ps, 14, NgramDrafter(), n_draft=6, tree=True) == ref


def test_model_drafter_tree_matches_greedy():
    cfg = LAYOUTS["mla_dense"]
    w = init_weights(cfg, seed=0)
    ps = prompts(cfg.vocab_size)
    ref = make(cfg, w).generate(ps, 10)
    draft = make(cfg, w, prefix_cache=True)
    eng = make(cfg, w)
    assert eng.generate_speculative(ps, 10, ModelDrafter(draft), n_draft=6, tree=True) == ref
    assert eng.stats["verify_steps"] == 3                    # the target's own chain: three of six drafts per step


def test_ngram_tree():
    d = NgramDrafter()
    toks, par = d.propose_tree([1, 2, 3, 9, 1, 2, 4, 1, 2], 4)
    # most recent (1, 2) -> 4 1 2; the one before -> 3 ...
    assert toks == [4, 1, 2, 3] and par == [0, 1, 2, 0]
    assert d.propose_tree([5, 6, 7], 3) == ([], [])


def test_sampling_is_reproducible_and_warm():
    cfg = LAYOUTS["mla"]
    w = init_weights(cfg, seed=0)
    ps = prompts(cfg.vocab_size)
    run = lambda seed, t, tree: make(cfg, w).generate_speculative(ps, 8, n_draft=4, tree=tree, temperature=t, seed=seed)
    assert run(1, 1.0, True) == run(1, 1.0, True)
    assert run(1, 1.0, True) != run(2, 1.0, True)
    assert all(len(o) == 8 for o in run(1, 1.0, False))
    assert run(1, 1e-4, True) == make(cfg, w).generate(ps, 8)     # nearly cold: the greedy tokens


def test_verify_tree_refusals():
    cfg = LAYOUTS["mla"]
    eng = make(cfg, init_weights(cfg, seed=0))
    r = eng.add_request([1, 2, 3])
    eng.prefill([r])
    with pytest.raises(ValueError, match="pending token"):
        eng.verify_tree([r], [([], [])])
    with pytest.raises(ValueError, match="one parent per node"):
        eng.verify_tree([r], [([1, 2], [-1])])
    with pytest.raises(ValueError, match="parent of node 1"):
        eng.verify_tree([r], [([1, 2], [-1, 1])])
    assert len(eng.verify_tree([r], [([5], [-1])])[0]) == 1


def test_failed_logits_are_reported():
    cfg = LAYOUTS["mla_dense"]
    eng = make(cfg, init_weights(cfg, seed=0))
    r = eng.add_request([1, 2, 3])
    eng.prefill([r])
    forward = eng.model.forward
    eng.model.forward = lambda fb, cache: forward(fb, cache) * float("nan")
    with pytest.raises(RuntimeError, match="not finite"):
        eng.verify_tree([r], [([5], [-1])])
