"""Sizes, inputs, plain forms and 64-bit definitions of the tree-speculation operators.

One step of speculative decoding drafts a small tree of tokens for every request and runs all of them through the
model at once.  Three operators belong to such a step:

* ``attend``: absorbed MLA / latent-MQA attention of every drafted node over its request's paged latent cache and over
  its own branch of the tree.
* ``verify``: the walk down the tree that accepts or rejects drafted tokens against the target's probabilities from
  given random numbers, and the token that follows the accepted path.
* ``commit``: the accepted nodes' cached rows, of every layer, moved to the positions that follow the context.

``own`` False: elementary torch operations in 32 bits; True: the calls of ``carbon_b200.ops.spec``.
"""
import math
import random

import torch

own = False


# ----------------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------------
def _attend(requests, context, nodes, heads, width=576, rows="bf16", page=64, sink=False, chain=False, ragged=True):
    return dict(op="attend", requests=requests, context=context, nodes=nodes, heads=heads, width=width, rows=rows,
                page=page, sink=sink, chain=chain, ragged=ragged)


def _verify(requests, nodes, vocab, drafts="probs", greedy=0.0, logits="fp32", chain=False, ragged=True):
    return dict(op="verify", requests=requests, nodes=nodes, vocab=vocab, drafts=drafts, greedy=greedy, logits=logits,
                chain=chain, ragged=ragged)


def _commit(requests, nodes, layers, row_bytes, page=64):
    return dict(op="commit", requests=requests, nodes=nodes, layers=layers, row_bytes=row_bytes, page=page)


def listed():
    return [
        # one interactive request with five drafts behind its last token, fp8 cache: the smallest call of a server
        dict(_attend(1, 700, 6, 128, rows="fp8", chain=True), name="attend one chain"),
        # the serving batch of the benchmark (32 requests near a context of 4096, five drafts each, fp8 cache)
        dict(_attend(32, 4096, 6, 128, rows="fp8", chain=True), name="attend serving batch"),
        # single tokens: plain decoding through the same call, bf16 cache
        dict(_attend(64, 2500, 1, 128), name="attend single tokens"),
        # trees of 24 nodes on a batch of mixed lengths, bf16 cache
        dict(_attend(12, 6000, 24, 128), name="attend trees"),
        # one rank's 16 heads of a tensor-parallel model on two very long contexts
        dict(_attend(2, 131072, 12, 16, ragged=False), name="attend long context"),
        # 512-wide rows (latent MQA) with per-head sinks, 16-token pages, odd sizes
        dict(_attend(7, 1999, 33, 64, width=512, page=16, sink=True), name="attend latent mqa"),
        # the largest: 32 requests, contexts up to 8192, trees of 32 nodes
        dict(_attend(32, 8192, 32, 128), name="attend wide trees"),
        # one request, five deterministic drafts (prompt lookup), the full vocabulary
        dict(_verify(1, 6, 129280, drafts="tokens", chain=True, ragged=False), name="verify one chain"),
        # the serving batch with trees drawn from a draft model's distributions
        dict(_verify(32, 12, 129280), name="verify trees"),
        # many requests of a smaller model, an odd vocabulary, bf16 logits, a third of them greedy
        dict(_verify(61, 16, 32003, drafts="tokens", greedy=0.33, logits="bf16"), name="verify mixed"),
        # one request's accepted rows in 61 layers of an fp8 cache
        dict(_commit(1, 6, 61, 656), name="commit one"),
        # a batch with wide trees, 61 layers of a bf16 cache
        dict(_commit(32, 24, 61, 1152), name="commit batch"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend"] * 6 + ["verify"] * 3 + ["commit"])
    if kind == "attend":
        while True:
            width = rng.choice([576, 576, 576, 512])
            c = _attend(_log(rng, 1, 64), _log(rng, 1, 131072), _log(rng, 1, 64), rng.choice([128, 128, 64, 32, 16, 5]),
                        width=width, rows=rng.choice(["bf16", "fp8"]), page=rng.choice([64, 64, 64, 128, 16, 24, 5]),
                        sink=rng.random() < 0.3, chain=rng.random() < 0.3, ragged=rng.random() < 0.8)
            rows = c["requests"] * c["context"]
            # cost, keys held, and the plain form's scores stay below the largest listed case's
            if rows <= 262144 and rows * c["nodes"] * c["heads"] <= 32 * 8192 * 32 * 128:
                return c
    if kind == "verify":
        while True:
            c = _verify(_log(rng, 1, 96), _log(rng, 1, 64), _log(rng, 500, 150000), drafts=rng.choice(["probs", "tokens"]),
                        greedy=rng.choice([0.0, 0.0, 0.3, 1.0]), logits=rng.choice(["fp32", "fp32", "bf16"]),
                        chain=rng.random() < 0.4, ragged=rng.random() < 0.8)
            if c["requests"] * c["nodes"] * c["vocab"] <= 32 * 16 * 129280:
                return c
    while True:
        c = _commit(_log(rng, 1, 96), _log(rng, 2, 64), rng.choice([61, 40, 4, 2]), rng.choice([656, 528, 1152, 1024]),
                    page=rng.choice([64, 64, 16]))
        if c["requests"] * c["layers"] <= 32 * 61:
            return c


# ----------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------
def _layout(case, seed):
    """Trees, contexts and page tables, as lists: what a server's scheduler holds.  The sizes belong to the case, the
    trees' shapes and the pages to the seed."""
    r = random.Random(13)
    B, n = case["requests"], case["nodes"]
    ragged = case.get("ragged", True)
    chain = case.get("chain", False)
    sizes = [r.randint(max(1, n // 2), n) if ragged else n for _ in range(B)]
    sizes[r.randrange(B)] = n
    top = case.get("context", 40)
    ctx = [r.randint(max(1, top // 2), top) if ragged else top for _ in range(B)]
    ctx[r.randrange(B)] = top
    r = random.Random(seed * 7919 + 13)
    parents = [[-1] + [i - 1 if chain or r.random() < 0.5 else r.randrange(i) for i in range(1, k)] for k in sizes]
    page = case.get("page", 64)
    need = [-(-(c + k) // page) for c, k in zip(ctx, sizes)]
    ids = list(range(1, sum(need) + 1))          # page 0 is a server's scratch page
    r.shuffle(ids)
    tables, at = [], 0
    for k in need:
        tables.append(ids[at:at + k])
        at += k
    return sizes, parents, ctx, tables, sum(need) + 1


def _quant_rows(x, width):
    """Rows [n, width] -> the fp8 cache row: e4m3 values of dims 0..255, 8 power-of-two scale bytes (one per 64 dims)
    and 8 zeros, e4m3 values of dims 256..511, then the last 64 dims of a 576-wide row in fp16."""
    n = x.shape[0]
    v = x[:, :512].reshape(n, 8, 64)
    amax = v.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax / 448.0)).clamp(-126, 127)
    q = (v / torch.exp2(e)).to(torch.float8_e4m3fn).view(torch.uint8).reshape(n, 512)
    s = (e.reshape(n, 8) + 127).to(torch.uint8)
    parts = [q[:, :256], s, torch.zeros_like(s), q[:, 256:]]
    if width == 576:
        parts.append(x[:, 512:].to(torch.float16).contiguous().view(torch.uint8))
    return torch.cat(parts, 1).contiguous()


def _expand_rows(rows, width, dtype):
    """Cached rows -> values in ``dtype`` (fp8 rows expanded; bf16 rows converted)."""
    if rows.dtype != torch.uint8:
        return rows.to(dtype)
    shape = rows.shape[:-1]
    q = torch.cat([rows[..., :256], rows[..., 272:528]], -1).view(torch.float8_e4m3fn).to(dtype)
    s = torch.exp2(rows[..., 256:264].to(dtype) - 127)
    v = (q.reshape(*shape, 8, 64) * s[..., None]).reshape(*shape, 512)
    if width == 576:
        v = torch.cat([v, rows[..., 528:].contiguous().view(torch.float16).to(dtype)], -1)
    return v


def _masks(parents):
    """Bit j of entry i: node i attends to node j (itself and its ancestors)."""
    out = []
    for i, p in enumerate(parents):
        out.append((1 << i) | (out[p] if p >= 0 else 0))
    return out


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed * 1000003 + 7)
    sizes, parents, ctx, tables, pages = _layout(case, seed)
    B, N = case["requests"], max(sizes)
    cu = [0]
    for k in sizes:
        cu.append(cu[-1] + k)
    T, page = cu[-1], case.get("page", 64)
    st = dict(case=case, B=B, N=N, T=T)
    node = torch.tensor([[i if i < k else -1 for i in range(N)] for k in sizes], device=dev)
    row = torch.tensor([[cu[b] + i if i < k else 0 for i in range(N)] for b, k in enumerate(sizes)], device=dev)
    st["there"], st["row"] = node >= 0, row
    st["flat"] = torch.tensor([b * N + i for b, k in enumerate(sizes) for i in range(k)], device=dev)
    st["parent"] = torch.tensor([p + [-2] * (N - len(p)) for p in parents], device=dev)
    st["ctx"] = torch.tensor(ctx, device=dev)
    P = max(len(t) for t in tables)
    st["tables"] = torch.tensor([t + [0] * (P - len(t)) for t in tables], device=dev)
    if own:
        from carbon_b200.ops.spec import TreePlan

        st["plan"] = TreePlan(tables, ctx, parents, page, n_heads=case.get("heads", 1), device=dev)

    if case["op"] == "attend":
        H, D = case["heads"], case["width"]
        # queries and latent rows of normalised activations; a few rows of every context draw most of the attention
        rows = torch.empty(pages * page, D, device=dev).normal_(generator=g)
        rows *= 0.7 + 0.6 * torch.rand(rows.shape[0], 1, device=dev, generator=g)
        rows = rows.to(torch.bfloat16)
        if case["rows"] == "fp8":
            st["cache"] = _quant_rows(rows.float(), D)
            q_type = torch.float16               # the model hands fp16 queries to an fp8 cache
        else:
            st["cache"], q_type = rows, torch.bfloat16
        st["q"] = torch.empty(T, H, D, device=dev).normal_(generator=g).to(q_type)
        st["sink"] = torch.empty(H, device=dev).normal_(generator=g) if case["sink"] else None
        st["scale"] = (192 if D == 576 else 512) ** -0.5
        sees = torch.zeros(B, N, N, dtype=torch.bool)
        for b, p in enumerate(parents):
            for i, m in enumerate(_masks(p)):
                for j in range(i + 1):
                    sees[b, i, j] = bool(m >> j & 1)
        st["sees"] = sees.to(dev)
        return st

    if case["op"] == "verify":
        V = case["vocab"]
        # target and draft logits that agree as well as a small model agrees with a large one
        base = torch.empty(T, V, device=dev).normal_(generator=g) * 5
        logits = base + 0.5 * torch.empty(T, V, device=dev).normal_(generator=g)
        draft = torch.softmax(base + 0.5 * torch.empty(T, V, device=dev).normal_(generator=g), -1)
        del base
        st["logits"] = logits.to(torch.bfloat16 if case["logits"] == "bf16" else torch.float32)
        # tokens of the children of each node: drawn from its draft distribution, or the draft's best ones in order
        width = max([1] + [p.count(i) for p in parents for i in range(len(p))])
        if case["drafts"] == "probs":
            kids = torch.multinomial(draft, width, replacement=True, generator=g)
            st["draft"] = draft
        else:
            kids = torch.topk(draft, width, dim=-1).indices
            st["draft"] = None
        src, rank = [], []
        for b, p in enumerate(parents):
            seen = {}
            for i, q in enumerate(p):
                src.append(cu[b] + max(q, 0))
                rank.append(seen.get(q, 0))
                seen[q] = rank[-1] + 1
        st["tokens"] = kids[torch.tensor(src, device=dev), torch.tensor(rank, device=dev).clamp(max=width - 1)].int()
        st["uniform"] = torch.rand(T, device=dev, generator=g)
        st["noise"] = torch.empty(B, V, device=dev).exponential_(generator=g)
        r = random.Random(seed + 5)
        st["temperature"] = torch.tensor([0.0 if r.random() < case["greedy"] else r.choice([0.7, 0.8, 1.0])
                                          for _ in range(B)], device=dev)
        return st

    L, W = case["layers"], case["row_bytes"]
    whole = torch.randint(0, 256, (L, pages * page, W), dtype=torch.uint8, device=dev, generator=g)
    # a list of per-layer caches, bf16 rows or raw fp8 rows (finite bf16 values: the exponent's top bit stays clear)
    if W in (1152, 1024):
        whole = (whole & 0xBF).view(torch.bfloat16)
    st["caches"] = list(whole.unbind(0))
    r = random.Random(seed + 9)
    path, count = [], []
    for p in parents:
        depth = [0] * len(p)
        for i in range(1, len(p)):
            depth[i] = depth[p[i]] + 1
        leaf = r.choice([i for i in range(len(p)) if depth[i] * 2 >= max(depth)])
        one = []
        while leaf >= 0:
            one.append(leaf)
            leaf = p[leaf]
        one.reverse()
        path.append(one + [-1] * (N - len(one)))
        count.append(len(one) - 1)
    st["path"] = torch.tensor(path, dtype=torch.int32, device=dev)
    st["count"] = torch.tensor(count, dtype=torch.int32, device=dev)
    if own:
        from carbon_b200.ops.spec import CacheRows

        st["handle"] = CacheRows(st["caches"])
    return st


# ----------------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------------
def run(st):
    op = st["case"]["op"]
    if own:
        from carbon_b200.ops import spec

        if op == "attend":
            return spec.tree_mla(st["q"], st["cache"], st["plan"], st["scale"], 512, sink=st["sink"])
        if op == "verify":
            v = spec.tree_verify(st["logits"], st["tokens"], st["plan"], st["uniform"], st["noise"],
                                 st["temperature"], draft_probs=st["draft"])
            return {"path": v.path, "accepted": v.n_accepted, "tokens": v.tokens, "logprobs": v.logprobs}
        spec.tree_commit(st["handle"], st["plan"], st["path"], st["count"])
        return st["caches"]
    return {"attend": _plain_attend, "verify": _plain_verify, "commit": _plain_commit}[op](st)


def _plain_attend(st):
    case, B, N = st["case"], st["B"], st["N"]
    H, D, page = case["heads"], case["width"], case["page"]
    pos = torch.arange(st["tables"].shape[1] * page, device="cuda")
    slots = (st["tables"][:, :, None] * page + torch.arange(page, device="cuda")).flatten(1)             # [B, L]
    keys = _expand_rows(st["cache"][slots], D, torch.float32)                                            # [B, L, D]
    q = st["q"][st["row"]].float().reshape(B, N * H, D)
    s = torch.bmm(q, keys.transpose(1, 2)).view(B, N, H, -1) * st["scale"]
    # prefix positions are seen by every node, tree positions by the node's own branch
    at = pos[None] - st["ctx"][:, None]                                                                  # [B, L]
    branch = torch.gather(st["sees"], 2, at.clamp(0, N - 1)[:, None].expand(B, N, -1)) & ((at >= 0) & (at < N))[:, None]
    see = (branch | (at < 0)[:, None]) & st["there"][:, :, None]                                         # [B, N, L]
    s = torch.where(see[:, :, None], s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    if st["sink"] is not None:
        top = torch.maximum(top, st["sink"].view(1, 1, H, 1))
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if st["sink"] is not None:
        total = total + torch.exp(st["sink"].view(1, 1, H, 1) - top)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.bmm(p.view(B, N * H, -1), keys[..., :512]).view(B, N, H, 512)
    return o.view(B * N, H, 512)[st["flat"]].to(torch.bfloat16)


def _plain_verify(st):
    B, N, V = st["B"], st["N"], st["case"]["vocab"]
    row, parent, there = st["row"], st["parent"], st["there"]
    each = torch.arange(B, device="cuda")
    temp = st["temperature"]
    cold = temp <= 0
    vocab = torch.arange(V, device="cuda")

    def target(node):
        """Probabilities [B, V] at each request's node, and the log-probabilities that are reported."""
        l = st["logits"][row[each, node]].float()
        scaled = l / torch.where(cold, 1.0, temp)[:, None]
        top = scaled.amax(-1, keepdim=True)
        e = torch.exp(scaled - torch.where(top == float("-inf"), 0.0, top))
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total > 0, total, 1.0)
        best = (vocab == torch.argmax(l, -1)[:, None]).float() * (total > 0)
        return torch.where(cold[:, None], best, p), scaled - top - torch.log(total)

    cur = torch.zeros(B, dtype=torch.long, device="cuda")
    left, logp = target(cur)
    path = torch.full((B, N), -1, dtype=torch.int32, device="cuda")
    tokens = torch.full((B, N), -1, dtype=torch.int32, device="cuda")
    logprobs = torch.zeros(B, N, device="cuda")
    path[:, 0] = 0
    count = torch.zeros(B, dtype=torch.long, device="cuda")
    for i in range(1, N):                        # a node's parent and older siblings come before it
        x = st["tokens"][row[:, i]].long()
        here = (parent[:, i] == cur) & there[:, i]
        if st["draft"] is not None:
            q = st["draft"][row[each, cur]]
        else:
            q = (vocab == x[:, None]).float()
        take = here & (st["uniform"][row[:, i]] * q[each, x] < left[each, x])
        if st["draft"] is not None:
            rest = (left - q).clamp(min=0)
        else:
            rest = torch.where(vocab == x[:, None], 0.0, left)
        mass = rest.sum(-1, keepdim=True)
        rest = torch.where(mass > 0, rest / torch.where(mass > 0, mass, 1.0), left)
        left = torch.where((here & ~take)[:, None], rest, left)
        # accepted: the node joins the path and its own distribution takes over
        slot = count.clamp(max=N - 2)
        tokens[each, slot] = torch.where(take, x.int(), tokens[each, slot])
        logprobs[each, slot] = torch.where(take, logp[each, x], logprobs[each, slot])
        count = count + take
        path[each, count] = torch.where(take, torch.full_like(cur, i).int(), path[each, count])
        cur = torch.where(take, i, cur)
        fresh, fresh_log = target(cur)
        left = torch.where(take[:, None], fresh, left)
        logp = torch.where(take[:, None], fresh_log, logp)
    # the race: the smallest noise / probability wins with its probability; without noise for greedy requests
    score = torch.where(left > 0, left / torch.where(cold[:, None], 1.0, st["noise"]), -1.0)
    best = torch.argmax(score, -1)
    ok = score[each, best] > 0
    tokens[each, count] = torch.where(ok, best, -1).int()
    logprobs[each, count] = torch.where(ok, logp[each, best], float("-inf"))
    return {"path": path, "accepted": count.int(), "tokens": tokens, "logprobs": logprobs}


def _plain_commit(st):
    page, N = st["case"]["page"], st["N"]
    k = torch.arange(N, device="cuda")
    live = (k[None] >= 1) & (k[None] <= st["count"][:, None])

    def slot(pos):
        return torch.gather(st["tables"], 1, pos // page) * page + pos % page

    # entries past the accepted path copy the root's row onto itself
    src = slot(st["ctx"][:, None] + torch.where(live, st["path"].long(), 0)).flatten()
    dst = slot(st["ctx"][:, None] + torch.where(live, k[None], 0)).flatten()
    for c in st["caches"]:
        c[dst] = c[src]
    return st["caches"]


# ----------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------------
def work(case):
    sizes, parents, ctx, tables, pages = _layout(case, 1)
    T = sum(sizes)
    if case["op"] == "attend":
        H, D = case["heads"], case["width"]
        row = 2 * D if case["rows"] == "bf16" else (656 if D == 576 else 528)
        keys = sum(c + k for c, k in zip(ctx, sizes))
        depth = []
        for p in parents:
            d = []
            for q in p:
                d.append(1 + (d[q] if q >= 0 else 0))
            depth.append(sum(d))
        pairs = sum(c * k + d for c, k, d in zip(ctx, sizes, depth))
        return {"bytes": keys * row + T * H * (2 * D + 1024), "flops": 2.0 * pairs * H * (D + 512)}
    if case["op"] == "verify":
        # rows off the walked path need not be read: the root's, and one more where there is a tree, are counted
        V, rows = case["vocab"], case["requests"] * min(2, case["nodes"])
        b = rows * V * (2 if case["logits"] == "bf16" else 4) + case["requests"] * V * 4 * (case["greedy"] < 1)
        if case["drafts"] == "probs":
            b += rows * V * 4
        return {"bytes": b, "flops": 4.0 * rows * V}
    moved = sum(max(1, len(p) // 4) for p in parents)        # accepted rows: about half a path's depth
    return {"bytes": 2.0 * moved * case["layers"] * case["row_bytes"], "flops": 0.0}


# ----------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """One request, one node at a time, from the definitions."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    sizes, parents, ctx, tables, _ = _layout(case, seed)
    if case["op"] == "attend":
        H, D, page = case["heads"], case["width"], case["page"]
        out, at = [], 0
        for n, p, c, t in zip(sizes, parents, ctx, tables):
            slots = torch.tensor([t[i // page] * page + i % page for i in range(c + n)], device="cuda")
            k = _expand_rows(st["cache"][slots], D, torch.float64)
            for i, m in enumerate(_masks(p)):
                sel = torch.tensor([j for j in range(n) if m >> j & 1], device="cuda", dtype=torch.long)
                kk = torch.cat([k[:c], k[c + sel]])
                s = st["q"][at + i].double() @ kk.T * st["scale"]
                if st["sink"] is not None:
                    w = torch.softmax(torch.cat([s, st["sink"].double()[:, None]], 1), 1)[:, :-1]
                else:
                    w = torch.softmax(s, 1)
                out.append(w @ kk[:, :512])
            at += n
        return torch.stack(out)
    if case["op"] == "verify":
        return _exact_verify(case, st, sizes, parents)
    if st["caches"][0].dtype == torch.uint8:
        return None                              # bytes are moved, nothing is computed
    page, moved = case["page"], [c.double() for c in st["caches"]]
    for b, (one, k) in enumerate(zip(st["path"].tolist(), st["count"].tolist())):
        at = [tables[b][(ctx[b] + i) // page] * page + (ctx[b] + i) % page for i in range(sizes[b])]
        for i in range(1, k + 1):
            for c in moved:
                c[at[i]] = c[at[one[i]]]
    return moved


def _exact_verify(case, st, sizes, parents):
    B, N = len(sizes), st["N"]
    path = torch.full((B, N), -1, dtype=torch.int32)
    tokens = torch.full((B, N), -1, dtype=torch.int32)
    logprobs = torch.zeros(B, N, dtype=torch.float64)
    count = torch.zeros(B, dtype=torch.int32)
    drafted, uniform = st["tokens"].tolist(), st["uniform"].double().tolist()
    at = 0
    for b, (n, par) in enumerate(zip(sizes, parents)):
        heat = float(st["temperature"][b])
        v, steps = 0, 0
        path[b, 0] = 0
        while True:
            l = st["logits"][at + v].double()
            lp = torch.log_softmax(l / (heat if heat > 0 else 1.0), 0)
            if heat > 0:
                r = lp.exp()
            else:
                r = torch.zeros_like(lp)
                r[int((l == l.max()).nonzero()[0])] = 1.0
            nxt = None
            for i in [j for j in range(n) if par[j] == v]:
                x = drafted[at + i]
                if st["draft"] is None:
                    q = torch.zeros_like(r)
                    q[x] = 1.0
                    without = r.clone()
                    without[x] = 0.0
                else:
                    q = st["draft"][at + v].double()
                    without = (r - q).clamp(min=0)
                if uniform[at + i] * float(q[x]) < float(r[x]):
                    nxt = i
                    break
                if float(without.sum()) > 0:
                    r = without / without.sum()
            if nxt is None:
                break
            tokens[b, steps], logprobs[b, steps] = x, lp[x]
            steps, v = steps + 1, nxt
            path[b, steps] = v
        race = r / (st["noise"][b].double() if heat > 0 else 1.0)
        win = int((race == race.max()).nonzero()[0])
        tokens[b, steps], logprobs[b, steps] = win, lp[win]
        count[b] = steps
        at += n
    return {"path": path, "accepted": count, "tokens": tokens, "logprobs": logprobs}
