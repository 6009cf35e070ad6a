"""Tree-speculation kernels against the definitions in 64 bits.

Attention tolerances: the output is rounded to bf16 (relative error at most 2^-9 each) and the softmax weights enter the
value product as 16-bit numbers (2^-9 each, averaging out over the keys), so the relative 2-norm error stays below
2^-9 + 2^-9 = 3.9e-3; 5e-3 is asserted.  A single value may be off by 2^-8 of itself plus the weights' share,
2^-8 of the row's largest value."""
import random

import pytest
import torch

from carbon_b200.ops import spec
from carbon_b200.ref import ops as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_plan(parents, ctx, page=64, heads=128, masks=None, seed=0, first_page=1):
    need = [-(-(c + len(p)) // page) for c, p in zip(ctx, parents)]
    ids = list(range(first_page, first_page + sum(need)))
    random.Random(seed).shuffle(ids)
    tables = []
    for k in need:
        tables.append(ids[:k])
        ids = ids[k:]
    return spec.TreePlan(tables, ctx, parents, page, n_heads=heads, device=DEV, masks=masks), \
        (first_page + sum(need)) * page


def tree(n, seed, chain=False):
    r = random.Random(seed)
    return [-1] + [i - 1 if chain or r.random() < 0.5 else r.randrange(i) for i in range(1, n)]


def rows_of(kv, D):
    return R.dequant_latent_fp8(kv, 512, D - 512, D == 576) if kv.dtype == torch.uint8 else kv.float()


def exact(q, kv, plan, scale, sink=None):
    D = q.shape[2]
    out = []
    masks = plan.mask.tolist()
    for b in range(plan.B):
        lo, hi = plan.cu_list[b], plan.cu_list[b + 1]
        if lo == hi:
            continue
        keys = rows_of(kv[torch.tensor(plan.slots(b), device=kv.device, dtype=torch.long)], D).double()
        out.append(R.tree_attention(q[lo:hi].double(), keys, plan.ctx_list[b], masks[lo:hi], scale, 512,
                                    None if sink is None else sink.double()))
    return torch.cat(out)


def close(got, want):
    got = got.double()
    assert bool(torch.isfinite(got).all())
    err = ((got - want).norm() / want.norm().clamp(min=1e-30)).item()
    assert err < 5e-3, err
    top = want.abs().amax(-1, keepdim=True)
    assert bool(((got - want).abs() <= 2 ** -8 * want.abs() + 2 ** -8 * top + 1e-30).all())


def inputs(plan, S, H, D, f8, seed=0, sink=False, peak=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kv = torch.randn(S, D, device=DEV, generator=g) * (0.5 + torch.rand(S, 1, device=DEV, generator=g))
    kv = R.quant_latent_fp8(kv, 512, 64, D == 576) if f8 else kv.to(torch.bfloat16)
    q = (peak * torch.randn(plan.T, H, D, device=DEV, generator=g)).to(torch.float16 if f8 else torch.bfloat16)
    return q, kv, (2 * torch.randn(H, device=DEV, generator=g) if sink else None)


SCALE = 192 ** -0.5
CASES = [
    # nodes per request, contexts, heads, width, fp8, page, sink
    ([1], [0], 128, 576, False, 64, False),
    ([1], [1], 16, 576, True, 64, True),
    ([6], [700], 128, 576, True, 64, False),
    ([1, 1, 1], [63, 64, 65], 128, 576, False, 64, False),
    ([2, 3, 1], [127, 128, 129], 128, 512, False, 64, True),
    ([7, 1, 33], [255, 0, 191], 64, 576, True, 64, True),
    ([64, 5], [100, 1000], 16, 576, False, 64, False),
    ([64], [64], 5, 512, True, 64, False),
    ([3, 0, 9], [40, 77, 300], 1, 576, False, 64, False),
    ([12, 4], [333, 1500], 32, 576, False, 16, False),
    ([12, 4], [333, 1500], 32, 576, True, 24, True),
    ([10, 17], [90, 411], 128, 512, False, 5, False),
    ([10, 17], [90, 411], 128, 512, True, 1, False),
    ([24, 31], [4000, 2500], 128, 576, False, 128, False),
    ([8], [9000], 16, 576, True, 64, False),
    ([1] * 40, [50 * i for i in range(40)], 128, 576, False, 64, False),
]


@pytest.mark.parametrize("n,ctx,H,D,f8,page,sink", CASES)
def test_tree_mla_against_64_bits(n, ctx, H, D, f8, page, sink):
    plan, S = make_plan([tree(k, i) if k else [] for i, k in enumerate(n)], ctx, page, H)
    q, kv, sk = inputs(plan, S, H, D, f8, seed=len(n) + ctx[0], sink=sink)
    close(spec.tree_mla(q, kv, plan, SCALE, sink=sk), exact(q, kv, plan, SCALE, sk))


@pytest.mark.parametrize("f8", [False, True])
def test_tree_mla_peaked_scores(f8):
    """Scores that grow along the context by hundreds (the running maximum moves in every tile)."""
    plan, S = make_plan([tree(5, 1), tree(3, 2)], [1000, 700], heads=128)
    q, kv, _ = inputs(plan, S, 128, 576, f8, seed=3, peak=4.0)
    if not f8:
        ramp = torch.linspace(0.1, 3.0, 1003, device=DEV)
        slots = torch.tensor(plan.slots(0), device=DEV)
        kv[slots[:1003]] = (kv[slots[:1003]].float() * ramp[:, None]).to(torch.bfloat16)
    close(spec.tree_mla(q, kv, plan, SCALE), exact(q, kv, plan, SCALE))


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("ctx", [0, 100])
def test_tree_mla_masks_that_leave_rows_empty(f8, ctx):
    masks = [[0, 2, 1, 0b1010, 0, 0b110000]]
    plan, S = make_plan([tree(6, 0)], [ctx], heads=16, masks=masks)
    for sink in (False, True):
        q, kv, sk = inputs(plan, S, 16, 576, f8, seed=4, sink=sink)
        got, want = spec.tree_mla(q, kv, plan, SCALE, sink=sk), exact(q, kv, plan, SCALE, sk)
        close(got, want)
        if ctx == 0:
            assert bool((got[[0, 4]] == 0).all())


@pytest.mark.parametrize("D,page", [(576, 64), (512, 64), (576, 24)])
@pytest.mark.parametrize("f8", [False, True])
def test_tree_mla_garbage_outside_the_mask(D, page, f8):
    """NaN and infinities in unwritten rows, in other requests' rows and in nodes of other branches do not reach a
    node that does not see them; a node that sees a NaN row is NaN."""
    parents = [[-1, 0, 0, 1, 2, 2], [-1, 0]]
    plan, S = make_plan(parents, [150, 70], page, 128)
    q, kv, _ = inputs(plan, S, 128, D, f8, seed=5)
    want = exact(q, kv, plan, SCALE)
    used = torch.zeros(S, dtype=torch.bool, device=DEV)
    used[torch.tensor(plan.slots(0) + plan.slots(1), device=DEV)] = True
    bad = torch.tensor(plan.slots(0)[152], device=DEV)                  # node 2 of request 0: seen by 2, 4, 5
    if f8:
        kv[~used] = 0x7F                                                # e4m3 NaN, largest scales, fp16 NaN
        kv[bad] = 0x7F
    else:
        kv[~used] = float("nan")
        kv[~used, ::2] = float("inf")
        kv[bad] = float("nan")
    got = spec.tree_mla(q, kv, plan, SCALE)
    clean = [0, 1, 3, 6, 7]
    close(got[clean], want[clean])
    assert bool(torch.isnan(got[[2, 4, 5]]).all())


def test_tree_mla_beyond_32_bit_offsets():
    """A cache of 4.6 GB: the pages lie past the 4 GiB boundary."""
    S = 4_000_000
    kv = torch.empty(S, 576, dtype=torch.bfloat16, device=DEV)
    plan, end = make_plan([tree(9, 3)], [500], heads=128, first_page=62400)
    assert end <= S
    q, part, _ = inputs(plan, 700, 128, 576, False, seed=6)
    slots = torch.tensor(plan.slots(0), device=DEV)
    kv[slots] = part[:509]
    close(spec.tree_mla(q, kv, plan, SCALE), exact(q, kv, plan, SCALE))


def test_tree_mla_repeats_bitwise_and_on_a_side_stream():
    plan, S = make_plan([tree(6, i) for i in range(5)], [900, 20, 3000, 0, 64], heads=128)
    q, kv, _ = inputs(plan, S, 128, 576, False, seed=7)
    a = spec.tree_mla(q, kv, plan, SCALE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = spec.tree_mla(q, kv, plan, SCALE)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b)


def test_tree_mla_strided_query_and_graph_capture():
    plan, S = make_plan([tree(6, 1)], [300], heads=16)
    q, kv, _ = inputs(plan, S, 32, 576, False, seed=8)
    part = q[:, ::2]                                                    # every second head: strided rows
    want = exact(part, kv, plan, SCALE)
    close(spec.tree_mla(part, kv, plan, SCALE), want)
    part = part.contiguous()
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        spec.tree_mla(part, kv, plan, SCALE)
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(g):
        out = spec.tree_mla(part, kv, plan, SCALE)
    g.replay()
    close(out, want)


def test_tree_mla_refusals():
    plan, S = make_plan([tree(2, 0)], [10], heads=16)
    q, kv, _ = inputs(plan, S, 16, 576, False)
    with pytest.raises(RuntimeError, match="D=576"):
        spec.tree_mla(q[:, :, :512].contiguous()[..., :448], kv, plan, SCALE)
    with pytest.raises(ValueError, match="heads"):
        spec.tree_mla(q[:, :8], kv, plan, SCALE)
    with pytest.raises(ValueError, match="slot"):
        spec.tree_mla(q, kv[:64], plan, SCALE)
    with pytest.raises(ValueError, match="width 576"):
        spec.tree_mla(q, kv[:, :512].contiguous(), plan, SCALE)
    with pytest.raises(ValueError, match="bfloat16"):
        spec.tree_mla(q, kv.float(), plan, SCALE)
    with pytest.raises(ValueError, match="not contiguous"):
        spec.tree_mla(q, torch.cat([kv, kv], 1)[:, :576], plan, SCALE)
    with pytest.raises(ValueError, match="sink"):
        spec.tree_mla(q, kv, plan, SCALE, sink=torch.zeros(3, device=DEV))
    empty = spec.TreePlan([], [], [], 64, n_heads=16, device=DEV)
    assert spec.tree_mla(q[:0], kv, empty, SCALE).shape == (0, 16, 512)


# ----------------------------------------------------------------------------------------------------------------------
# verification
# ----------------------------------------------------------------------------------------------------------------------
def verify_inputs(parents, V, seed, probs, dtype=torch.float32, temps=(0.8,), spread=4.0):
    g = torch.Generator().manual_seed(seed)
    T, B = sum(len(p) for p in parents), len(parents)
    base = torch.randn(T, V, generator=g) * spread
    logits = (base + torch.randn(T, V, generator=g)).to(dtype)
    draft = torch.softmax(base + torch.randn(T, V, generator=g), -1)
    src = []
    at = 0
    for p in parents:
        src += [at + max(0, x) for x in p]
        at += len(p)
    tok = torch.multinomial(draft[src], 1, generator=g)[:, 0].int() if T else torch.zeros(0, dtype=torch.int32)
    temp = torch.tensor([temps[i % len(temps)] for i in range(B)])
    return dict(logits=logits, tokens=tok, uniforms=torch.rand(T, generator=g),
                noise=torch.empty(B, V).exponential_(generator=g), temperature=temp,
                draft_probs=draft if probs else None)


def check_verify(parents, kw):
    plan, _ = make_plan(parents, [0] * len(parents))
    v = spec.tree_verify(plan=plan, **{k: x.to(DEV) if x is not None else None for k, x in kw.items()})
    v = spec.TreeVerdict(*[x.cpu() for x in v])
    at = 0
    for b, p in enumerate(parents):
        n = len(p)
        if n == 0:
            assert v.n_accepted[b] == -1 and bool((v.path[b] == -1).all()) and bool((v.tokens[b] == -1).all())
            continue
        path, toks, lps = R.tree_verify(kw["logits"][at:at + n].double(), kw["tokens"][at:at + n], p,
                                        kw["uniforms"][at:at + n].double(), kw["noise"][b].double(),
                                        float(kw["temperature"][b]),
                                        None if kw["draft_probs"] is None else kw["draft_probs"][at:at + n].double())
        k = len(path)
        assert v.path[b].tolist() == path + [-1] * (plan.N - k), b
        assert v.tokens[b].tolist() == toks + [-1] * (plan.N - k), b
        assert v.n_accepted[b] == k - 1
        # fp32 logits of magnitude <= 40 over temperatures >= 0.5: 80 * 2^-23 = 1e-5, and as much for the sum
        torch.testing.assert_close(v.logprobs[b, :k].double(), torch.tensor(lps, dtype=torch.float64), rtol=0, atol=2e-5)
        assert bool((v.logprobs[b, k:] == 0).all())
        at += n
    return v


@pytest.mark.parametrize("V", [1, 2, 31, 1000, 4099, 32003, 129280])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tree_verify_against_64_bits(V, probs, dtype):
    parents = [tree(1, 0), tree(6, 1, chain=True), tree(12, 2), [], [-1] + [0] * 7, tree(9, 4), tree(64, 5)]
    check_verify(parents, verify_inputs(parents, V, V + probs, probs, dtype, temps=(0.8, 1.0, 0.0, 1.3)))


def test_tree_verify_many_requests():
    parents = [tree(1 + i % 13, i) for i in range(150)]
    v = check_verify(parents, verify_inputs(parents, 3001, 9, True, temps=(1.0, 0.6)))
    assert 0 < int((v.n_accepted > 0).sum()) < 150


@pytest.mark.parametrize("requests,V,probs,dtype", [
    (16, 20011, False, torch.float32), (20, 32003, True, torch.bfloat16), (48, 20500, False, torch.bfloat16),
    (86, 4100, True, torch.float32), (70, 700, False, torch.float32), (70, 700, False, torch.bfloat16)])
def test_tree_verify_shares_of_the_vocabulary(requests, V, probs, dtype):
    """Numbers of CTAs per request that are no powers of two, shares that end inside a 16-byte piece, short rows."""
    parents = [tree(1 + i % 6, i, chain=i % 2 == 0) for i in range(requests)]
    check_verify(parents, verify_inputs(parents, V, requests, probs, dtype, temps=(0.8, 0.0)))


def test_tree_verify_unaligned_bf16_rows():
    """bf16 logits that start at an odd column of a wider tensor whose other columns hold NaN."""
    parents = [tree(6, i, chain=True) for i in range(3)]
    kw = verify_inputs(parents, 70001, 4, False, torch.bfloat16, temps=(0.9, 0.0, 1.0))
    plan, _ = make_plan(parents, [0] * 3)
    on = {k: x.to(DEV) if x is not None else None for k, x in kw.items()}
    a = spec.tree_verify(plan=plan, **on)
    for first in (1, 2, 7):
        wide = torch.full((18, 70011), float("nan"), device=DEV, dtype=torch.bfloat16)
        wide[:, first:first + 70001] = on["logits"]
        b = spec.tree_verify(plan=plan, **{**on, "logits": wide[:, first:first + 70001]})
        assert torch.equal(a.path, b.path) and torch.equal(a.tokens, b.tokens)
        # the rows' pieces start elsewhere, so sums round differently: 2e-5 as against 64 bits
        torch.testing.assert_close(a.logprobs, b.logprobs, rtol=0, atol=2e-5)


def test_tree_verify_duplicate_and_unknown_tokens():
    """Siblings with the same token, and tokens outside the vocabulary (never accepted), without draft probabilities."""
    parents = [[-1, 0, 0, 0, 0]] * 8
    kw = verify_inputs(parents, 50, 3, False, spread=1.0)
    kw["tokens"] = torch.tensor([0, 7, 7, 9, 7] * 8, dtype=torch.int32)
    check_verify(parents, kw)
    plan, _ = make_plan(parents, [0] * 8)
    kw["tokens"] = torch.tensor([0, -5, 50, 2 ** 31 - 1, -2 ** 31] * 8, dtype=torch.int32)
    v = spec.tree_verify(plan=plan, **{k: x.to(DEV) if x is not None else None for k, x in kw.items()})
    assert bool((v.n_accepted == 0).all()) and bool((v.tokens[:, 0] >= 0).all())


def test_tree_verify_masked_rows():
    """Logits of -inf (a token filter), of the type's lowest value, and rows with nothing left."""
    parents = [[-1, 0, 0], [-1, 0], [-1, 0], [-1, 0]]
    kw = verify_inputs(parents, 500, 5, False, temps=(1.0,))
    kw["logits"][0:3, 20:] = float("-inf")
    kw["logits"][3:5, :499] = torch.finfo(torch.float32).min
    kw["logits"][5:7] = float("-inf")
    kw["temperature"][3] = 0.0
    kw["logits"][7:9] = float("-inf")
    v = check_verify(parents, kw)
    assert v.tokens[1, 0] == 499 and v.tokens[2, 0] == -1 and v.tokens[3, 0] == -1


def test_tree_verify_row_stride():
    """Logits that are columns of a wider tensor (a vocabulary padded for the projection)."""
    parents = [tree(6, 1), tree(4, 2)]
    kw = verify_inputs(parents, 1001, 6, True)
    wide = torch.full((10, 1024), 99.0, device=DEV)
    wide[:, :1001] = kw["logits"].to(DEV)
    plan, _ = make_plan(parents, [0, 0])
    on = {k: x.to(DEV) for k, x in kw.items()}
    a = spec.tree_verify(plan=plan, **on)
    on["logits"] = wide[:, :1001]
    b = spec.tree_verify(plan=plan, **on)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_tree_verify_target_distribution():
    """40,000 requests with the same target row: the first emitted token is distributed as the target (each
    frequency within 5 standard deviations, 5 * sqrt(0.25 / 40000) = 0.0125)."""
    g = torch.Generator(device=DEV).manual_seed(2)
    V, B, n = 12, 40000, 4
    p = torch.softmax(torch.randn(V, device=DEV, generator=g), -1)
    q = torch.softmax(torch.randn(V, device=DEV, generator=g), -1)
    plan = spec.TreePlan([[1]] * B, [0] * B, [[-1, 0, 0, 0]] * B, 64, device=DEV)
    tok = torch.multinomial(q, B * n, replacement=True, generator=g).int()
    v = spec.tree_verify(p.log().expand(B * n, V).contiguous(), tok, plan, torch.rand(B * n, device=DEV, generator=g),
                         torch.empty(B, V, device=DEV).exponential_(generator=g), torch.ones(B, device=DEV),
                         draft_probs=q.expand(B * n, V).contiguous())
    freq = torch.bincount(v.tokens[:, 0].long(), minlength=V).double() / B
    assert bool(((freq - p.double()).abs() < 0.0125).all())
    assert bool((v.n_accepted <= 1).all())


def test_tree_verify_refusals():
    plan, _ = make_plan([[-1, 0]], [0])
    ok = dict(logits=torch.zeros(2, 6, device=DEV), tokens=torch.zeros(2, dtype=torch.int32, device=DEV), plan=plan,
              uniforms=torch.zeros(2, device=DEV), noise=torch.ones(1, 6, device=DEV),
              temperature=torch.zeros(1, device=DEV))
    spec.tree_verify(**ok)
    for name, bad, what in (("logits", torch.zeros(2, 6, device=DEV, dtype=torch.float16), "fp32 or bf16"),
                            ("logits", torch.zeros(6, 2, device=DEV).t(), "column stride"),
                            ("tokens", torch.zeros(2, dtype=torch.int64, device=DEV), "tokens must be"),
                            ("uniforms", torch.zeros(2), "uniforms must be"),
                            ("noise", torch.ones(1, 6, device=DEV, dtype=torch.float64), "noise must be"),
                            ("draft_probs", torch.zeros(2, 6, device=DEV, dtype=torch.bfloat16), "draft_probs")):
        with pytest.raises(ValueError, match=what):
            spec.tree_verify(**{**ok, name: bad})


# ----------------------------------------------------------------------------------------------------------------------
# commit
# ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("page", [64, 7])
def test_tree_commit_moves_rows(page):
    parents = [[-1, 0, 0, 2, 2, 4], [-1, 0], [-1], [], tree(64, 3, chain=True), [-1, 0, 1, 1, 3, 3, 5, 6, 7, 7]]
    ctx = [60, 5, 0, 9, 130, 1]
    plan, S = make_plan(parents, ctx, page)
    g = torch.Generator().manual_seed(0)
    caches = [torch.randint(0, 256, (S, w), dtype=torch.uint8, generator=g) for w in (656, 528, 12, 4)]
    caches += [torch.randn(S, w, generator=g).to(torch.bfloat16) for w in (576, 512, 128, 2, 6)]
    caches += [torch.arange(S, dtype=torch.int32)]
    N = plan.N
    paths = [[0, 2, 4, 5], [0], [0], [], [0] + list(range(1, 64)), [0, 1, 3, 5, 6, 7, 9]]
    path = torch.tensor([p + [-1] * (N - len(p)) for p in paths], dtype=torch.int32)
    n = torch.tensor([len(p) - 1 for p in paths], dtype=torch.int32)
    want = [c.clone() for c in caches]
    for b, p in enumerate(paths):
        at = plan.slots(b)[ctx[b]:]
        for k in range(1, len(p)):
            for c in want:
                c[at[k]] = c[at[p[k]]]
    dev = [c.to(DEV) for c in caches]
    spec.tree_commit(spec.CacheRows(dev), plan, path.to(DEV), n.to(DEV))
    for got, w in zip(dev, want):
        assert torch.equal(got.cpu().view(torch.uint8), w.view(torch.uint8))


def test_tree_commit_refusals():
    plan, S = make_plan([[-1, 0]], [0])
    cache = torch.zeros(S, 8, device=DEV)
    rows = spec.CacheRows([cache])
    path, n = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    spec.tree_commit(rows, plan, path, n)
    with pytest.raises(ValueError, match="path"):
        spec.tree_commit(rows, plan, path.long(), n)
    with pytest.raises(ValueError, match="n_accepted"):
        spec.tree_commit(rows, plan, path, n.cpu())
    with pytest.raises(ValueError, match="slot"):
        spec.tree_commit(spec.CacheRows([cache[:64]]), plan, path, n)
    with pytest.raises(ValueError, match="one device"):
        spec.CacheRows([cache, cache.cpu()])


# ----------------------------------------------------------------------------------------------------------------------
# the engine's step
# ----------------------------------------------------------------------------------------------------------------------
def engine_cfg(kind):
    from carbon_b200.config import small_gpu_config

    cfg = small_gpu_config().replace(n_layers=2, n_routed_experts=8, n_activated_experts=2, vocab_size=2048)
    if kind == "dense":
        return cfg.replace(index_n_heads=0, index_topk=0)
    if kind == "dense_fp8":
        return cfg.replace(index_n_heads=0, index_topk=0, kv_fp8=True, attn_sink=True)
    if kind == "latent":
        return cfg.replace(attn_kind="latent_mqa", index_n_heads=0, index_topk=0, attn_sink=True)
    return cfg                                                # DSA


@pytest.mark.parametrize("kind", ["dense", "dense_fp8", "latent", "dsa"])
def test_engine_tree_step_matches_row_verification(kind):
    """One tree step of three requests against the same nodes as decode rows (each node's branch appended to its own
    copy of the context): the logits differ by the kernels' rounding only.  Both paths round the attention output to
    bf16 (2^-9) and run the same fp8 GEMMs on it, whose own rounding (2^-4 relative per input) can flip single inputs
    by one step; 5 % of the logits' norm bounds that over two layers (flips of router choices are excluded by the
    comparison of the median row)."""
    from carbon_b200.engine.engine import Engine
    from carbon_b200.models.weights import WeightSource
    from carbon_b200.ref.model import init_weights

    cfg = engine_cfg(kind)
    w = init_weights(cfg, seed=0)
    g = torch.Generator().manual_seed(1)
    ps = [torch.randint(0, cfg.vocab_size, (k,), generator=g).tolist() for k in (70, 131, 300)]
    trees = [([5, 6, 7, 8], [-1, 0, 0, 1]), ([9], [-1]), ([1, 2, 3, 4, 5], [-1, 0, 1, 1, 2])]
    eng = Engine(cfg, device="cuda", source=WeightSource(cfg, state=w), num_pages=96, page_size=64)
    rows = []
    for p, (toks, par) in zip(ps, trees):
        for i in range(len(toks)):
            branch = []
            k = i
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
        seen["plan"] = fb.tree
        return seen["logits"]

    eng.model.forward = keep
    out = eng.verify_tree(reqs, trees)
    seen["plan"].check()
    want = torch.stack(rows)
    err = ((seen["logits"].float() - want).norm(dim=-1) / want.norm(dim=-1)).sort().values
    assert err[len(err) // 2] < 0.05, err
    # the walk agrees with the step's own logits, and the committed branch continues like a plain context
    best = seen["logits"].float().argmax(-1).tolist()
    assert out[1] == [best[4]]
    eng.model.forward = forward
    nxt = eng.decode(reqs, [o[-1] for o in out])
    assert bool(torch.isfinite(nxt).all())
    for r, p, o, (toks, _) in zip(reqs, ps, out, trees):
        assert r.out == [toks[0]] + o


@pytest.mark.parametrize("kind", ["dense", "dsa"])
def test_engine_tree_speculation_gpu(kind):
    """Greedy trees drafted by the target itself: every chain token is accepted and the sequence is the target's own
    greedy continuation (the draft engine and the target run the same kernels)."""
    from carbon_b200.engine.engine import Engine
    from carbon_b200.engine.spec import ModelDrafter
    from carbon_b200.models.weights import WeightSource
    from carbon_b200.ref.model import init_weights

    cfg = engine_cfg(kind)
    w = init_weights(cfg, seed=0)
    g = torch.Generator().manual_seed(2)
    ps = [torch.randint(0, cfg.vocab_size, (k,), generator=g).tolist() for k in (50, 200)]
    mk = lambda **kw: Engine(cfg, device="cuda", source=WeightSource(cfg, state=w), num_pages=64, page_size=64, **kw)
    eng = mk()
    out = eng.generate_speculative(ps, 8, ModelDrafter(mk()), n_draft=6, tree=True)
    assert all(len(o) == 8 for o in out)
    warm = mk().generate_speculative(ps, 8, n_draft=4, tree=True, temperature=1.0, seed=3)
    again = mk().generate_speculative(ps, 8, n_draft=4, tree=True, temperature=1.0, seed=3)
    assert warm == again
