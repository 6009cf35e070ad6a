"""Speculative decoding over trees of drafted tokens: attention, verification and the commit of the accepted branch.

One step runs, for every request, a small tree of drafted tokens (node 0 is the pending token, every other node
continues its parent) through the model in one forward.  ``TreePlan`` holds the step's layout on the device; the three
operators take it:

* ``tree_mla``     absorbed MLA / latent-MQA attention of all nodes: each node sees its request's whole context and its
                   own branch of the tree.  The cached rows are read once per 128 query rows (nodes x heads), not once
                   per node (``sparse_mla`` gathers every row's key list again).
* ``tree_verify``  the walk down the tree that accepts drafted tokens against the target's probabilities from given
                   random numbers, and the token that follows (temperature 0: greedy agreement).
* ``tree_commit``  the accepted nodes' cached rows, in every cache of a ``CacheRows``, moved behind the context.

Conventions: the rows of a request's nodes are consecutive (``plan.cu``); node i of request b writes its cache rows at
position ``ctx[b] + i`` of the request's page table.  Everything runs on the current stream, allocates from the caching
allocator and neither waits for the device nor reads from it.  The oracle is ``ref.ops.tree_attention`` /
``tree_verify``; CPU tensors use it.  The reference verifies chains of drafts as ordinary decode rows
(``king_v10/bundle_v9/dec/gemm_tables.py:51``, ``dec/cuda_vattn.py:4654``).
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence

import torch

from ..ref import ops as R
from ._ext import ext

_ROW_BYTES = {576: 656, 512: 528}      # an fp8 cache row (ref.ops.latent_fp8_row_bytes)
_STAGE_BYTES = 512 << 20               # of the dense rows of one call: 465,000 keys of 576 dims
MAX_NODES = 64           # nodes of one request's tree: one bit each in a node's mask


_CLUSTERS = {}


def _clusters(device: torch.device) -> int:
    """CTA pairs of the attention kernel that the device runs at once."""
    if device not in _CLUSTERS:
        with torch.cuda.device(device):
            _CLUSTERS[device] = ext().tree_mla_clusters()
        if not _CLUSTERS[device]:
            raise RuntimeError(f"tree_mla: the attention kernel does not fit on {device}")
    return _CLUSTERS[device]


class TreePlan:
    """Layout of one tree step.  page_tables[b] lists request b's pages (at least ctx[b] + n_b positions), ctx[b] its
    cached tokens, parents[b][i] the parent of node i (-1 for the root, node 0; parents come before children).
    ``masks``: per request one integer per node, bit j = node i attends to node j; by default each node's ancestors
    and itself.  Requests without nodes are allowed.  A plan serves every layer and operator of its step."""

    def __init__(self, page_tables: Sequence[Sequence[int]], ctx: Sequence[int], parents: Sequence[Sequence[int]],
                 page_size: int, n_heads: int = 1, device="cuda", masks: Optional[Sequence[Sequence[int]]] = None):
        self.device = torch.device(device)
        cuda = self.device.type == "cuda"
        if cuda and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.page_size, self.n_heads = int(page_size), int(n_heads)
        self.ctx_list, self.tables_list, self.parents_list = list(ctx), page_tables, parents
        code = -1
        if cuda and masks is None:
            code, host, self._counts, meta = ext().tree_plan(page_tables, self.ctx_list, parents, self.page_size,
                                                             self.n_heads, _clusters(self.device))
        if code:                            # other devices, given masks, and arguments that do not fit (raises)
            host, meta = self._lists(masks)
        w, T, self.N, P, self.max_page = meta
        self.n = [len(p) for p in parents]
        B = self.B = len(self.n)
        self.T = T
        self._host = host
        dev = host.to(self.device, non_blocking=True)
        self._work = dev[:w]
        self.mask = dev[w:w + 2 * T].view(torch.int64)
        self.status = dev[-1:]              # error code of a device-side wait that ran out (0: none)
        at = self._at = w + 2 * T
        out = []
        for k in (B + 1, B, T, T, T, T, B * P):
            out.append(dev[at:at + k])
            at += k
        self.cu, self.ctx, self.req, self.parent, self.pos, self.slot, self.table = out
        self.table = self.table.view(B, P)

    def _lists(self, masks):
        """The plan's lists in one buffer, as the native builder lays them out: (buffer, lengths)."""
        page_tables, ctx, parents, page_size = self.tables_list, self.ctx_list, self.parents_list, self.page_size
        B = len(parents)
        if len(page_tables) != B or len(ctx) != B or (masks is not None and len(masks) != B):
            raise ValueError("TreePlan: page_tables, ctx, parents (and masks) need one entry per request")
        if page_size < 1 or self.n_heads < 1:
            raise ValueError("TreePlan: page_size and n_heads must be positive")
        cu, req, par, pos, slot, bits = [0], [], [], [], [], []
        for b, (p, c, tab) in enumerate(zip(parents, ctx, page_tables)):
            k = len(p)
            if k > MAX_NODES:
                raise ValueError(f"TreePlan: request {b} has {k} nodes, at most {MAX_NODES} are supported")
            if c < 0 or (c + k + page_size - 1) // page_size > len(tab):
                raise ValueError(f"TreePlan: request {b} has pages for {len(tab) * page_size} positions, its context "
                                 f"and nodes need {c + k}")
            if any(pg < 0 for pg in tab):
                raise ValueError(f"TreePlan: request {b} has a negative page")
            if any((pg + 1) * page_size > 2 ** 31 - 1 for pg in tab):
                raise ValueError(f"TreePlan: request {b} has a page past 2^31 slots")
            depth = []
            for i, q in enumerate(p):
                if not (q == -1 if i == 0 else 0 <= q < i):
                    raise ValueError(f"TreePlan: request {b}: the parent of node {i} must be an earlier node "
                                     "(-1 for node 0 only)")
                depth.append(depth[q] + 1 if i else 0)
            m = R.tree_masks(p) if masks is None else [int(x) for x in masks[b]]
            if len(m) != k or any(x < 0 or x >> k for x in m):
                raise ValueError(f"TreePlan: request {b} needs one mask of {k} bits per node")
            bits += [x - (1 << 64) if x >> 63 else x for x in m]
            cu.append(cu[-1] + k)
            req += [b] * k
            par += p
            pos += [c + d for d in depth]
            slot += [tab[(c + i) // page_size] * page_size + (c + i) % page_size for i in range(k)]
        P = max([len(t) for t in page_tables] + [1])
        flat = []
        for tab in page_tables:
            flat += list(tab)
            flat += [0] * (P - len(tab))
        work, self._counts = torch.zeros(0, dtype=torch.int32), []
        cuda = self.device.type == "cuda"
        if cuda and cu[-1]:
            got = ext().tree_plan(page_tables, ctx, parents, page_size, self.n_heads, _clusters(self.device))
            work, self._counts = got[1][:got[3][0]], got[2]
        host = torch.cat([work, torch.tensor(bits, dtype=torch.int64).view(torch.int32),
                          torch.tensor(cu + list(ctx) + req + par + pos + slot + flat + [0], dtype=torch.int32)])
        top = max((pg for tab in page_tables for pg in tab), default=-1)
        return (host.pin_memory() if cuda else host), (work.numel(), cu[-1], max((len(p) for p in parents), default=0),
                                                       P, top)

    @property
    def cu_list(self) -> List[int]:
        """First node row of each request, and the number of rows."""
        return self._host[self._at:self._at + self.B + 1].tolist()

    @property
    def pos_list(self) -> List[int]:
        """Position of each node in its sequence (its depth behind the context)."""
        at = self._at + 2 * self.B + 1 + 2 * self.T
        return self._host[at:at + self.T].tolist()

    def check(self, status: Optional[int] = None) -> None:
        """Raise if a kernel of this plan gave up a wait.  Reads ``status`` from the device unless the caller has."""
        code = int(self.status) if status is None else status
        if code:
            raise RuntimeError(f"tree_mla: device status {code}: a bounded wait ran out")

    def slots(self, b: int, n: Optional[int] = None) -> List[int]:
        """Cache slots of request b's first n positions (default: its context and all its nodes)."""
        ps, tab = self.page_size, self.tables_list[b]
        n = self.ctx_list[b] + self.n[b] if n is None else n
        return [tab[i // ps] * ps + i % ps for i in range(n)]

    def node_slots(self) -> List[int]:
        """Cache slot of every node row (``slot`` on the device)."""
        at = self._at + 2 * self.B + 1 + 3 * self.T
        return self._host[at:at + self.T].tolist()

    def _check(self, what: str, slots: int):
        if (self.max_page + 1) * self.page_size > slots:
            raise ValueError(f"{what}: the plan's pages reach slot {(self.max_page + 1) * self.page_size - 1}, the "
                             f"cache holds {slots}")


def _need(what: str, t: torch.Tensor, dev: int, dtype) -> None:
    """dev: a CUDA device's index."""
    if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous {dtype} on cuda:{dev}, got {t.dtype} on {t.device}"
                         f"{'' if t.is_contiguous() else ' (not contiguous)'}")


def _aligned(what: str, t: torch.Tensor) -> None:
    """Rows are read 16 bytes at a time (row sizes are multiples of 16): an address off that grid would fault."""
    if t.data_ptr() % 16:
        raise ValueError(f"{what} must start on a 16-byte boundary (address modulo 16: {t.data_ptr() % 16})")


def _launched(code: int, what: str) -> None:
    if code:
        raise RuntimeError(f"{what}: CUDA error {code} at launch")


def _stage_rows(counts: Sequence[int], f8: bool, page_size: int, D: int) -> int:
    """Dense rows that a call expands its whole key tiles to before the attention (0: it does not).

    Whole key tiles that TMA cannot take from the cache as they lie (fp8 rows, small pages) are fed by the kernel's warps
    (4.0 us a tile and CTA pair), or expanded to dense rows first (2.0 us a tile then, and 2.8 us of every pair's time per
    staged tile; a launch): worth it from two row tiles per key tile and a few tiles per pair on.  32 requests near 4096,
    6 nodes of 128 heads: 204 us fed, 148 us staged; one node: 62 us fed, 85 us staged; 1 request of 700, 6 nodes: 19.3 us
    fed, 25.0 us staged.  Not past _STAGE_BYTES of dense rows: they are 1.76 times the fp8 cache rows, once per request even
    of pages that requests share, in the middle of a step on a device whose cache may fill it (fed past it: 1.25 times the
    time at 128 requests of 4096 keys and 6 nodes, 1.4 times with 24 nodes)."""
    pairs, tiles, work = counts[0], counts[4], counts[5]
    if not (f8 or page_size % 64) or not tiles or work < 2 * tiles or work < 4 * pairs:
        return 0
    return tiles * 128 if tiles * 128 * D * 2 <= _STAGE_BYTES else 0


def tree_mla(q: torch.Tensor, kv: torch.Tensor, plan: TreePlan, scale: float, d_latent: int = 512,
             sink: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the plan's nodes over the paged latent cache: q [T, H, D], kv [S, D] bf16 (or the fp8 cache rows,
    uint8 [S, row_bytes], with q in fp16; q is converted), D = 576 (MLA) or 512 (latent MQA) -> [T, H, 512] bf16.
    On a GPU kv is contiguous and starts on a 16-byte boundary.  sink [H]: per-head attention-sink logit.  A node that
    sees no key gives zeros."""
    T, H, D = q.shape
    f8 = kv.dtype == torch.uint8
    if T != plan.T:
        raise ValueError(f"tree_mla: q has {T} rows, the plan {plan.T} nodes")
    plan._check("tree_mla", kv.shape[0])
    if not scale > 0:
        raise ValueError(f"tree_mla: scale must be positive, got {scale}")
    if sink is not None and sink.shape != (H,):
        raise ValueError(f"tree_mla: sink has shape {tuple(sink.shape)}, expected {(H,)}")
    if q.is_cuda:
        if D not in (576, 512) or d_latent != 512:
            raise RuntimeError("tree_mla: the kernel needs D=576 (512 latent + 64 RoPE key) or D=512 (latent MQA) and "
                               "d_latent=512")
        if H != plan.n_heads:
            raise ValueError(f"tree_mla: q has {H} heads, the plan was made for {plan.n_heads}")
        dev = plan.device.index
        if q.get_device() != dev:
            raise ValueError(f"tree_mla: q is on {q.device}, the plan on {plan.device}")
        _need("tree_mla: kv", kv, dev, torch.uint8 if f8 else torch.bfloat16)
        if kv.dim() != 2 or kv.shape[1] != (_ROW_BYTES[D] if f8 else D):
            raise ValueError(f"tree_mla: kv of shape {tuple(kv.shape)} does not hold rows for width {D}")
        _aligned("tree_mla: kv", kv)
        want = torch.float16 if f8 else torch.bfloat16
        qk = q if q.dtype is want and q.is_contiguous() else q.to(want).contiguous()
        if qk.data_ptr() % 16:                           # the tensor map needs it
            qk = qk.clone()
        if sink is not None:
            _need("tree_mla: sink", sink, dev, torch.float32)
        out = torch.empty(T, H, 512, dtype=torch.bfloat16, device=q.device)
        if T:
            parts = plan._counts[3]
            rows = _stage_rows(plan._counts, f8, plan.page_size, D)
            staged = torch.empty(rows * D, dtype=want, device=q.device) if rows else None
            buf = torch.empty(parts * 128 * 514, dtype=torch.float32, device=q.device) if parts else None
            _launched(ext().tree_mla(qk, kv, plan.cu, plan.ctx, plan.table, plan.mask, plan.page_size, plan._work,
                                     plan._counts, buf, staged, float(scale), sink, plan.status, out), "tree_mla")
        return out
    out = torch.zeros(T, H, d_latent)
    mla = D > d_latent
    cu = plan.cu_list
    for b in range(plan.B):
        lo, hi = cu[b], cu[b + 1]
        rows = kv[torch.tensor(plan.slots(b), dtype=torch.long)]
        rows = R.dequant_latent_fp8(rows, d_latent, D - d_latent if mla else 0, mla) if f8 else rows.float()
        out[lo:hi] = R.tree_attention(q[lo:hi].float(), rows, plan.ctx_list[b], plan.mask[lo:hi].tolist(), scale,
                                      d_latent, sink)
    return out


class TreeVerdict(NamedTuple):
    """Outcome of ``tree_verify``, N = the largest tree's nodes: path [B, N] the accepted nodes (the root first),
    n_accepted [B] how many drafted nodes were accepted, tokens [B, N] the accepted tokens and then the next one,
    logprobs [B, N] their log-probabilities under the target at the request's temperature (at 1 when greedy).
    path and tokens are padded with -1, logprobs with 0.  A request without nodes has n_accepted -1."""

    path: torch.Tensor
    n_accepted: torch.Tensor
    tokens: torch.Tensor
    logprobs: torch.Tensor


def _check_verify(logits, tokens, plan, uniforms, noise, temperature, draft_probs) -> None:
    """Raise for the first argument of tree_verify that does not fit."""
    T, B, V = plan.T, plan.B, logits.shape[-1]
    for name, t, shape in (("logits", logits, (T, V)), ("tokens", tokens, (T,)), ("uniforms", uniforms, (T,)),
                           ("noise", noise, (B, V)), ("temperature", temperature, (B,)),
                           ("draft_probs", draft_probs, (T, V))):
        if t is not None and t.shape != shape:
            raise ValueError(f"tree_verify: {name} has shape {tuple(t.shape)}, expected {shape}")
    if logits.device != plan.device:
        raise ValueError(f"tree_verify: logits are on {logits.device}, the plan on {plan.device}")
    if plan.device.type != "cuda":
        return
    if logits.dtype not in (torch.float32, torch.bfloat16) or not 0 < V < 1 << 31 or (T and logits.stride(1) != 1):
        raise ValueError(f"tree_verify: logits must be fp32 or bf16 with a unit column stride, got {logits.dtype}, "
                         f"strides {logits.stride()}")
    for name, t, dtype in (("tokens", tokens, torch.int32), ("uniforms", uniforms, torch.float32),
                           ("noise", noise, torch.float32), ("temperature", temperature, torch.float32),
                           ("draft_probs", draft_probs, torch.float32)):
        if t is not None:
            _need(f"tree_verify: {name}", t, plan.device.index, dtype)


def tree_verify(logits: torch.Tensor, tokens: torch.Tensor, plan: TreePlan, uniforms: torch.Tensor,
                noise: torch.Tensor, temperature: torch.Tensor, draft_probs: Optional[torch.Tensor] = None
                ) -> TreeVerdict:
    """Accept or reject the drafted tokens (``ref.ops.tree_verify`` states the rule).  logits [T, V] fp32 or bf16 (unit
    column stride): the target's logits at every node; tokens [T] int32: every node's token (the root's is not
    tested); uniforms [T] fp32 in [0, 1): one per node; noise [B, V] fp32: Exp(1) variates; temperature [B] fp32 (0 =
    greedy); draft_probs [T, V] fp32: row t = the distribution that node t's children were drawn from (independent
    draws), None = certain proposals (prompt lookup, a draft model's best tokens).  The emitted tokens are distributed
    as the target's own samples."""
    B, N = plan.B, plan.N
    if logits.is_cuda and plan.device.type == "cuda":
        out = torch.empty(B * (3 * N + 1), dtype=torch.int32, device=plan.device)
        code, path, n, toks, lp = ext().tree_verify(logits, tokens, plan.cu, plan.parent, N, uniforms, noise,
                                                    temperature, draft_probs, out)
        if code == -1:
            _check_verify(logits, tokens, plan, uniforms, noise, temperature, draft_probs)
        _launched(code, "tree_verify")
        return TreeVerdict(path, n, toks, lp)
    _check_verify(logits, tokens, plan, uniforms, noise, temperature, draft_probs)
    v = TreeVerdict(torch.full((B, N), -1, dtype=torch.int32), torch.full((B,), -1, dtype=torch.int32),
                    torch.full((B, N), -1, dtype=torch.int32), torch.zeros(B, N))
    cu = plan.cu_list
    for b in range(B):
        lo, hi = cu[b], cu[b + 1]
        if lo == hi:
            continue
        path, toks, lps = R.tree_verify(logits[lo:hi].float(), tokens[lo:hi], plan.parents_list[b], uniforms[lo:hi],
                                        noise[b], float(temperature[b]),
                                        draft_probs[lo:hi] if draft_probs is not None else None)
        v.path[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
        v.tokens[b, :len(toks)] = torch.tensor(toks, dtype=torch.int32)
        v.logprobs[b, :len(lps)] = torch.tensor(lps)
        v.n_accepted[b] = len(path) - 1
    return v


class CacheRows:
    """The caches whose rows move together: tensors [S, ...] (one row per slot, any row size that is a multiple of 4
    bytes), contiguous, on one device and starting on a 4-byte boundary.  Holds the tensors and, on a GPU, the table of their addresses."""

    def __init__(self, caches: Sequence[torch.Tensor]):
        self.caches = [c for c in caches if c is not None]
        if not self.caches:
            raise ValueError("CacheRows: no caches")
        first = self.caches[0]
        self.device = first.device
        self.slots = min(c.shape[0] for c in self.caches)
        rows = []
        for c in self.caches:
            nbytes = c.numel() // max(1, c.shape[0]) * c.element_size()
            if c.device != first.device or not c.is_contiguous() or nbytes % 4 or not nbytes:
                raise ValueError("CacheRows: caches must be contiguous, on one device and have rows of a multiple of "
                                 "4 bytes")
            if c.data_ptr() % 4:
                raise ValueError("CacheRows: caches must start on a 4-byte boundary")
            rows += [c.data_ptr(), nbytes]
        self.max_row = max(rows[1::2])
        self.wide = all(x % 16 == 0 for x in rows)
        table = torch.tensor(rows, dtype=torch.int64).view(-1, 2)
        self._host = table.pin_memory() if first.is_cuda else table
        self.table = self._host.to(first.device, non_blocking=True)


def tree_commit(rows: CacheRows, plan: TreePlan, path: torch.Tensor, n_accepted: torch.Tensor) -> None:
    """Move the accepted branch's cache rows behind the context, in place: for k = 1 .. n_accepted[b], the row of node
    path[b, k] goes to position ctx[b] + k (node k's old row).  path [B, N] and n_accepted [B] as ``tree_verify``
    returns them."""
    if path.shape != (plan.B, plan.N) or n_accepted.shape != (plan.B,):
        raise ValueError(f"tree_commit: path {tuple(path.shape)} and n_accepted {tuple(n_accepted.shape)}, expected "
                         f"{(plan.B, plan.N)} and {(plan.B,)}")
    plan._check("tree_commit", rows.slots)
    if rows.device.type == "cuda":
        if rows.device != plan.device:
            raise ValueError(f"tree_commit: the caches are on {rows.device}, the plan on {plan.device}")
        _need("tree_commit: path", path, plan.device.index, torch.int32)
        _need("tree_commit: n_accepted", n_accepted, plan.device.index, torch.int32)
        if plan.N > 1:
            _launched(ext().tree_commit(rows.table, rows.max_row, rows.wide, plan.cu, plan.ctx, plan.table,
                                        plan.page_size, path, n_accepted), "tree_commit")
        return
    for b in range(plan.B):
        s = plan.slots(b)[plan.ctx_list[b]:]
        for k in range(1, int(n_accepted[b]) + 1):
            for c in rows.caches:
                c[s[k]] = c[s[int(path[b, k])]]
