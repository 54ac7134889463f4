"""Sequences that share pages: a paged cache with reference counts, and a decoder that serves
many samples of one prompt from it.

``SharedPagedKVCache`` is a ``PagedKVCache`` whose sequences take pages from one pool: a fork
shares the sealed blocks and copies the tail, a free gives pages back, a compaction brings the
pages in use to the pool's front (nsn_b200.pages).  Page 0 names no page.  Its decode step over
a ``share`` plan attends to a common prefix once for all its sequences (prefix_attention) and to
each sequence's own blocks and tail with the cache's decode kernels, joined by their
log-sum-exps.

``SharedPromptDecoder`` runs a looped model that way: one prompt through prompt_attention, its
cache forked to every sequence, then decode steps.  The reference runs one sequence at a time
through caches of its own (experiments/ac08/source/loop_kv_ac08_attention.py:46-96).
"""
from __future__ import annotations

import weakref

import numpy as np
import torch

from . import _lib as L
from . import pages as P
from . import primitives as w
from .kernel import decode_attention
from .looped import PagedLoopedDecoder
from .paged import PagedKVCache, block_record_pools, group_record_pools
from .prefix import prefix_attention
from .prompt import prompt_attention


class SharedPrefix:
    """Which sequences of a cache share which leading pages, laid out for its step_shared
    (made by SharedPagedKVCache.share; valid until a fork, free, prefill, import or compaction of
    it, from when on step_shared refuses the plan).

    ``own_table`` is a copy of the block table's entries behind the prefixes; step_shared brings it
    up to date when pages were assigned since (by any step, a seal, extend or reserve)."""

    def __init__(self, cache, groups):
        batch, dev = cache.batch, cache.device
        self.cache, self.held = weakref.ref(cache), cache.held
        table = cache.block_table.cpu().numpy()  # the one host read, when the plan is made
        first, n_pages, order, offsets = np.zeros(batch, np.int64), [], [], [0]
        for seqs in groups:
            rows = table[seqs]
            n = int(cache.host_blocks[seqs].min())
            same = (rows[:, :n] == rows[0, :n]).all(axis=0) & (rows[0, :n] > 0)
            n = n if same.all() else int(np.argmin(same))
            first[seqs] = n
            n_pages.append(n)
            order += list(seqs)
            offsets.append(len(order))
        order += [b for b in range(batch) if b not in set(order)]
        wide = max(n_pages + [1])
        pages = np.zeros((max(1, len(groups)), wide), np.int32)
        for g, seqs in enumerate(groups):
            pages[g, :n_pages[g]] = table[seqs[0], :n_pages[g]]
        put = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(dev)
        self.pages, self.n_pages = put(pages), put(n_pages or [0])
        self.row_offsets, self.row_index = put(offsets if groups else [0, 0]), put(order)
        self.max_rows = max([len(s) for s in groups] + [1])
        self.first = put(first)
        at = first[:, None] + np.arange(cache.max_blocks)[None]
        self.own_at = torch.from_numpy(np.minimum(at, cache.max_blocks - 1)).to(dev)
        self.own_table = torch.empty_like(cache.block_table)  # each row's entries behind the prefix
        self.own_blocks = torch.empty_like(cache.n_blocks)
        q_shape = (batch, cache.hq, w.DIM)
        self.o_part = torch.empty(q_shape, dtype=torch.float32, device=dev)
        self.lse_part = torch.empty(q_shape[:2], dtype=torch.float32, device=dev)
        self.lse = torch.empty(q_shape[:2], dtype=torch.float32, device=dev)
        self.ws = torch.empty(max(16, L.load().nsnkv_prefix_attn_workspace_bytes(
            batch, self.pages.shape[0], cache.hq, cache.h, wide)), dtype=torch.uint8, device=dev)
        self.refresh(cache)

    def refresh(self, cache):
        torch.gather(cache.block_table, 1, self.own_at, out=self.own_table)
        self.table_epoch = cache.table_epoch


class SharedPagedKVCache(PagedKVCache):
    """A PagedKVCache over a pool of ``pages`` pages (page 0 excepted) that its sequences share.

    INT3 or INT5 caches with hq / h <= 8 (the block-record layout), ``restore_rounding`` "k" or
    "exact".  Every sequence keeps one page reserved for its next block; when the pool runs out
    the status word gets NSNKV_ST_CAPACITY and the block that finds no page is lost, which
    ``check`` reports.  Pages held: sealed blocks, each once however many sequences share it,
    and the reserved ones.
    """

    def __init__(self, batch: int, h: int, max_blocks: int, pages: int, bits: int = 3, dtype=torch.float16,
                 device="cuda", hq: int | None = None, restore_rounding: str = "k"):
        w.require(pages > batch, "shared cache pages: at least one per sequence beside page 0")
        super().__init__(batch, h, max_blocks, bits=bits, dtype=dtype, device=device, hq=hq,
                         restore_rounding=restore_rounding, pages=pages)
        w.require(self.records is not None, "shared cache: INT3 or INT5 block records, hq / h <= 8")
        self.page_refs = torch.zeros(pages, dtype=torch.int32, device=self.device)
        self.page_refs[0] = 1
        self.table_epoch = 0  # counts the calls that may have assigned pages
        self.held = 0  # counts the calls that change what sequences hold other than by appending to them
        self.replayed = False  # a graph's replays assign pages too, without the host
        self.reserve()

    def _capturing(self):
        return L.capturing(self.device.index)

    # ------------------------------------------------------------ pages
    def _seqs(self, seqs, what):
        seqs = [int(b) for b in ([seqs] if isinstance(seqs, (int, np.integer)) else seqs)]
        w.require(all(0 <= b < self.batch for b in seqs), f"{what}: sequence numbers")
        return seqs

    def _dev(self, seqs):
        return torch.tensor(seqs, dtype=torch.int32, device=self.device)

    def reserve(self, seqs=None, ahead: int = 1):
        """Pages for the next ``ahead`` blocks of every sequence, or of sequence ``seqs``."""
        rows = slice(None) if seqs is None else slice(seqs, seqs + 1)
        P.reserve_pages(self.block_table[rows], self.n_blocks[rows], self.page_refs, ahead, self.status)
        self.table_epoch += 1
        self.replayed = self.replayed or self._capturing()

    def fork(self, src, dst):
        """Sequences ``dst`` become copies of sequence(s) ``src`` (one for all, or one each): the
        sealed pages shared, the tail copied, what dst held given back."""
        dst = self._seqs(dst, "fork")
        src = self._seqs(src, "fork")
        src = src * len(dst) if len(src) == 1 else src
        w.require(len(src) == len(dst) and len(set(dst)) == len(dst) and not set(src) & set(dst),
                  "fork: distinct targets, none of them a source")
        if not dst:
            return
        P.fork_sequences(self.block_table, self.n_blocks, self.tail_len, self.page_refs, self.k_tail, self.v_tail,
                         self._dev(src), self._dev(dst), self.status)
        self.host_blocks[dst] = self.host_blocks[src]
        self.host_tail[dst] = self.host_tail[src]
        self.held += 1
        self.reserve()

    def free(self, seqs):
        """Sequences give their pages back and are empty (one page stays reserved for each)."""
        seqs = self._seqs(seqs, "free")
        if not seqs:
            return
        P.free_sequences(self.block_table, self.n_blocks, self.tail_len, self.page_refs, self._dev(seqs), self.status)
        self.host_blocks[seqs] = 0
        self.host_tail[seqs] = 0
        self.held += 1
        self.reserve()

    def compact(self) -> torch.Tensor:
        """Bring the pages in use to the pool's front; returns their number (device int32 [1])."""
        self.held += 1
        self.table_epoch += 1
        return P.compact_pages([self.records, self.k_pool["norm"], self.v_pool["norm"]], self.block_table,
                               self.page_refs, table_out=self.block_table, refs_out=self.page_refs,
                               status=self.status)[2]

    # ------------------------------------------------------------ loading
    def _put(self, b, n, records, k_norm, v_norm):
        pages = self.block_table[b, self.host_blocks[b]:self.host_blocks[b] + n].long()
        self.records[:, pages] = records
        self.k_pool["norm"][:, pages] = k_norm
        self.v_pool["norm"][:, pages] = v_norm

    def _native(self, k, v, what):
        w.require(k.shape == v.shape and k.ndim == 3 and k.shape[0] == self.h and k.shape[2] == w.DIM, f"{what} shape")
        w.require(k.shape[1] < w.BLOCK or k.device == v.device == self.device, f"{what}: K and V on the cache's device")

    def extend(self, b: int, k: torch.Tensor, v: torch.Tensor):
        """Append native K/V [h, T, 128] to sequence b, whose tail is empty: T // 64 blocks are
        sealed, T % 64 tokens become the tail."""
        self._native(k, v, "extend")
        w.require(self.host_tail[b] == 0, "extend: the sequence's tail is not empty")
        n, t = k.shape[1] // w.BLOCK, k.shape[1] % w.BLOCK
        w.require(self.host_blocks[b] + n <= self.max_blocks, "extend exceeds max_blocks")
        self.reserve(b, min(n + 1, self.max_blocks))
        if n:
            records, kp, vp = block_record_pools(self.h, n, self.bits, self.device)
            for src, pool in ((k, kp), (v, vp)):
                x = src[:, :n * w.BLOCK].reshape(self.h, n, w.BLOCK, w.DIM).to(self.dtype)
                w.encode_blocks(x, self.bits, out=pool, out_row_stride=n, out_offset=0, check=False)
            self._put(b, n, records, kp["norm"], vp["norm"])
        if t:
            self.k_tail[b, :, :t].copy_(k[:, n * w.BLOCK:])
            self.v_tail[b, :, :t].copy_(v[:, n * w.BLOCK:])
        self._advance(b, n, t)

    def _advance(self, b, n, t):
        self.host_blocks[b] += n
        self.host_tail[b] = t
        self.n_blocks[b] = int(self.host_blocks[b])
        self.tail_len[b] = t
        self.reserve(b)

    def prefill(self, b: int, k: torch.Tensor, v: torch.Tensor):
        """Load sequence b from native K/V [h, T, 128] (what it held is given back)."""
        self._native(k, v, "prefill")
        w.require(k.shape[1] // w.BLOCK <= self.max_blocks, "prefill exceeds max_blocks")
        self.free([b])
        self.extend(b, k, v)

    def import_groups(self, b: int, kg, kt, vg, vt):
        """Load sequence b from the reference's layout (see PagedKVCache.import_groups)."""
        n = self._import_sizes(kg, kt, vg, vt)[0]
        if n:
            dev = lambda g: dict(g, codes=g["codes"].to(self.device), metas=tuple(m.to(self.device) for m in g["metas"]))
            records, kp, vp = group_record_pools(dev(kg), dev(vg), self.bits)
        kt, vt = (x[0].to(self.device, self.dtype) for x in (kt, vt))
        self.free([b])  # nothing is refused from here on
        self.reserve(b, min(n + 1, self.max_blocks))
        if n:
            self._put(b, n, records, kp["norm"], vp["norm"])
        self._advance(b, n, 0)
        self.extend(b, kt, vt)

    # ------------------------------------------------------------ decode
    def share(self, groups) -> SharedPrefix:
        """A plan for step_shared: in each group (a list of sequences) the leading pages that all
        of its sequences hold are attended to once.  Reads the block table back once."""
        groups = [self._seqs(g, "share") for g in groups]
        flat = [b for g in groups for b in g]
        w.require(all(groups) and len(set(flat)) == len(flat), "share: disjoint groups of sequences")
        return SharedPrefix(self, groups)

    def _after_seal(self):
        # a captured step replays with other counters: it always looks for pages
        if not self.host_tail.all() or self._capturing():
            self.reserve()

    def seal(self, pending_append: int = 1):
        super().seal(pending_append)
        self._after_seal()

    def step(self, q, k_new, v_new, out=None, attn_event=None):
        o = super().step(q, k_new, v_new, out=out, attn_event=attn_event)
        self._after_seal()
        return o

    def step_host(self, host_in, host_out, done_event=None):
        o = super().step_host(host_in, host_out, done_event)
        self._after_seal()
        return o

    def step_shared(self, plan: SharedPrefix, q, k_new, v_new, out=None):
        """``step`` with the plan's prefixes attended to once: append (k_new, v_new)
        [batch, h, 128], attend with q [batch, hq, 128] over prefix, own blocks and tail, seal.
        Prefix blocks are K- and V-rounded to the cache dtype as the bridge rounds them; own
        blocks follow ``restore_rounding``.  A graph that captured this call ends with its plan."""
        w.require(plan.cache() is self and plan.held == self.held,
                  "step_shared plan: of this cache, and made after its last fork, free, prefill, import and compaction")
        if ((self.host_blocks >= self.max_blocks) & (self.host_tail + 1 >= w.BLOCK)).any():
            L.check(L.ERR_TOO_LARGE, "step_shared")  # as step: the tail must keep a free row
        o = self.out if out is None else out
        if plan.table_epoch != self.table_epoch or self.replayed or self._capturing():
            plan.refresh(self)
        torch.sub(self.n_blocks, plan.first, out=plan.own_blocks)
        decode_attention(
            q, self.k_pool, self.v_pool, h=self.h, bits=self.bits, blk_stride_head=self.pages, blk_stride_page=1,
            n_blocks=plan.own_blocks, max_blocks=self.max_blocks, k_tail=self.k_tail, v_tail=self.v_tail,
            tail_stride_seq=self.h * w.BLOCK, tail_stride_head=w.BLOCK, tail_len=self.tail_len,
            max_tail=w.BLOCK - 1, block_table=plan.own_table, k_new=k_new, v_new=v_new, out=o, out_f32=plan.o_part,
            lse=plan.lse_part, status=self.status, ws=self.ws, blk_bytes=self.blk_bytes,
            exact=self.restore_rounding == "exact")
        prefix_attention(q, self.records, plan.pages, plan.n_pages, bits=self.bits, row_offsets=plan.row_offsets,
                         row_index=plan.row_index, max_rows=plan.max_rows, o_part=plan.o_part,
                         lse_part=plan.lse_part, out=o, lse=plan.lse, status=self.status, ws=plan.ws)
        self.seal(1)
        return o

    def check(self):
        st = int(self.status.item())
        if st & (L.ST_CAPACITY | L.ST_PAGE):
            raise w.ContractError("shared cache: no page for a block (the pool is exhausted, or a replay went past "
                                  "max_blocks)" if st & L.ST_CAPACITY
                                  else "shared cache: a page number outside the pool")
        super().check()


class SharedPromptDecoder(PagedLoopedDecoder):
    """A PagedLoopedDecoder whose sequences are samples of one prompt: the prompt runs once
    (prompt_attention), its cached blocks are shared by every sequence, and a decode step
    attends to them once for the whole batch.  ``pages``: pool pages per cache; the default
    holds max_tokens for every sequence apart, a shared prompt of n blocks needs n and each
    sequence's own blocks, one page reserved for each and page 0."""

    def __init__(self, model, batch: int, max_tokens: int, restore_rounding: str = "k", pages: int | None = None):
        self._pages = pages
        super().__init__(model, batch, max_tokens, restore_rounding)
        self.plans = None

    def _new_cache(self, restore_rounding):
        pages = self._pages or self.batch * self.max_blocks + 1
        return SharedPagedKVCache(self.batch, self.h, self.max_blocks, pages, bits=3, dtype=self.dtype,
                                  device=self.device, hq=self.hq, restore_rounding=restore_rounding)

    def _prefill_layer(self, layer, h, cos, sin, cache):
        attn, (_, T, _) = layer.self_attn, h.shape
        x = layer.input_layernorm(h)
        q = attn.q_proj(x).view(1, T, self.hq, self.head_dim).transpose(1, 2)
        k = attn.k_proj(x).view(1, T, self.h, self.head_dim).transpose(1, 2)
        v = attn.v_proj(x).view(T, self.h, self.head_dim)
        q, k = self.rope(q, k, cos, sin)
        o, _ = prompt_attention(q[0].transpose(0, 1), k[0].transpose(0, 1), v, self._cu, T, status=cache.status)
        cache.prefill(0, k[0], v.transpose(0, 1))
        cache.fork(0, range(1, self.batch))
        h = h + attn.o_proj(o.reshape(1, T, self.hq * self.head_dim))
        return h + layer.mlp(layer.post_attention_layernorm(h))

    @torch.no_grad()
    def prefill(self, ids: torch.Tensor) -> torch.Tensor:
        """The prompt's ids [P], for every sequence -> last-token logits [vocab]."""
        ids = ids.reshape(1, -1).to(self.device)
        n = ids.shape[1]
        if self.length:
            raise ValueError("SharedPromptDecoder.prefill: into empty caches")
        if n < 1 or n + 1 > 64 * (self.max_blocks - 1):
            raise ValueError("SharedPromptDecoder.prefill: the prompt exceeds max_tokens")
        self._cu = torch.tensor([0, n], dtype=torch.int32, device=self.device)
        logits = self._prefill_forward(ids, torch.arange(n, device=self.device)[None])[0]
        self.plans = {id(c): c.share([range(self.batch)]) for c in self.caches}
        self.length = n
        return logits

    def _attend(self, cache, q, k, v):
        return cache.step_shared(self.plans[id(cache)], q, k, v)
