"""Cases that time the shared-prompt operators: each in a plain torch form and as the library's call.

Three operators of serving a batch whose sequences start from one prompt:

  prompt  nsn_b200.prompt.prompt_attention: causal attention over whole prompts, packed one
          after another, grouped heads, (out, log-sum-exp) per row;
  prefix  nsn_b200.prefix.prefix_attention: attention of many query rows over a sealed INT3 /
          INT5 prefix that they share, K and V restored and rounded to the cache dtype as the
          bridge restores them, merged with each row's attention over its own tokens;
  pages   nsn_b200.pages.fork_sequences / compact_pages: forking sequences of a paged cache and
          compacting its page pool.

``own`` chooses what ``run`` calls: False, elementary torch operations in fp32 rounded once at
the end; True, the library.  ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK, DIM = 64, 128
SCALE = 1.0 / math.sqrt(DIM)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
OUTLIERS = [3, 37, 71, 105]  # K channels x8, as in the workloads' K


# ---------------------------------------------------------------------------------- cases
def listed():
    return [
        # three short chat turns prefilled together: a few tokens each, MHA; launch latency counts
        {"name": "prompt-short", "op": "prompt", "seqs": 3, "tokens": 59, "ragged": True, "hq": 16, "h": 16,
         "dtype": "fp16", "fused": True},
        # the looped decoder's prefill of one (loop, layer): 4 prompts of 2048 tokens, 16 MHA heads
        {"name": "prompt-looped", "op": "prompt", "seqs": 4, "tokens": 8192, "ragged": False, "hq": 16, "h": 16,
         "dtype": "fp16", "fused": False},
        # a ragged bf16 batch of prompts of odd lengths, GQA 32:8, read from the fused projection
        {"name": "prompt-ragged", "op": "prompt", "seqs": 9, "tokens": 9001, "ragged": True, "hq": 32, "h": 8,
         "dtype": "bf16", "fused": True},
        # one prompt of the batched workload's longest context, GQA 32:8
        {"name": "prompt-long", "op": "prompt", "seqs": 1, "tokens": 16384, "ragged": False, "hq": 32, "h": 8,
         "dtype": "fp16", "fused": False},
        # four samples of one short system prompt (8 blocks), GQA 32:8: latency
        {"name": "prefix-short", "op": "prefix", "groups": 1, "rows": 4, "blocks": 8, "bits": 3, "hq": 32, "h": 8,
         "dtype": "fp16"},
        # a decode step of 64 sequences that share an 8192-token prompt, GQA 32:8
        {"name": "prefix-batch", "op": "prefix", "groups": 1, "rows": 64, "blocks": 128, "bits": 3, "hq": 32, "h": 8,
         "dtype": "fp16"},
        # samples of one 131008-token INT5 document, GQA 64:8
        {"name": "prefix-long", "op": "prefix", "groups": 1, "rows": 8, "blocks": 2047, "bits": 5, "hq": 64, "h": 8,
         "dtype": "fp16"},
        # new turns (1501 prompt tokens in all) after three cached system prompts, bf16
        {"name": "prefix-continue", "op": "prefix", "groups": 3, "rows": 1501, "blocks": 96, "bits": 3, "hq": 32,
         "h": 8, "dtype": "bf16"},
        # one prompt forked into three more samples
        {"name": "fork-few", "op": "fork", "batch": 4, "sources": 1, "targets": 3, "max_blocks": 40, "h": 8,
         "dtype": "fp16"},
        # a beam step of the 64-sequence batch: 8 survivors refill the other 56 slots
        {"name": "fork-batch", "op": "fork", "batch": 64, "sources": 8, "targets": 56, "max_blocks": 300, "h": 8,
         "dtype": "fp16"},
        # compacting the small pool of a 4-sequence cache after one sequence left
        {"name": "compact-few", "op": "compact", "batch": 4, "max_blocks": 40, "pages": 161, "live": 97, "moves": 24,
         "h": 8, "bits": 3},
        # compacting the 64-sequence batch's pool when half of its pages came free
        {"name": "compact-batch", "op": "compact", "batch": 64, "max_blocks": 300, "pages": 19201, "live": 9600,
         "moves": 4800, "h": 8, "bits": 3},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prefix", "prefix", "fork", "compact"])
    h, g = rng.choice([(8, 4), (16, 1), (8, 8), (8, 4), (2, 2), (3, 6)])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "prompt":
        seqs = _log(rng, 1, 16)
        longest = int(16384 * math.sqrt(32.0 / (h * g) / seqs) / 1.5)  # bounds the plain form's scores
        tokens = max(seqs, _log(rng, 32, min(longest, 16384) * max(1, seqs // 2)))
        return {"op": op, "seqs": seqs, "tokens": tokens, "ragged": seqs > 1, "hq": h * g, "h": h, "dtype": dtype,
                "fused": rng.random() < 0.5}
    if op == "prefix":
        rows = _log(rng, 1, 1500)
        blocks = _log(rng, 1, max(1, min(2047, 2047 * 64 // (rows * g))))
        return {"op": op, "groups": min(rows, rng.choice([1, 1, 2, 3, 5])), "rows": rows, "blocks": blocks,
                "bits": rng.choice([3, 3, 5]), "hq": h * g, "h": h, "dtype": dtype}
    if op == "fork":
        batch = _log(rng, 2, 64)
        sources = rng.randint(1, max(1, batch // 2))
        return {"op": op, "batch": batch, "sources": sources, "targets": rng.randint(1, batch - sources),
                "max_blocks": _log(rng, 3, 300), "h": h, "dtype": dtype}
    batch, max_blocks, bits = _log(rng, 1, 64), _log(rng, 4, 256), rng.choice([3, 5])
    pages = batch * max_blocks + 1
    live = rng.randint(max(2, pages // 4), max(2, (3 * pages) // 4))
    most = 4800 if bits == 3 else 3000
    return {"op": op, "batch": batch, "max_blocks": max_blocks, "pages": pages, "live": live,
            "moves": rng.randint(1, min(most, live - 1, pages - live)), "h": min(h, 8), "bits": bits}


# --------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)


def _lengths(n, total, ragged, gen):
    """n positive lengths that sum to total: equal ones, or spread from one token to long ones."""
    if n == 1:
        return [total]
    if not ragged:
        return [total // n + (1 if i < total % n else 0) for i in range(n)]
    weight = [math.exp(3.0 * i / (n - 1)) for i in range(n)]
    order = torch.randperm(n, generator=gen, device="cuda").tolist()
    got = [1 + int((total - n) * w / sum(weight)) for w in weight]
    got[-1] += total - sum(got)
    got[0], got[-1] = 1, got[-1] + got[0] - 1
    return [got[i] for i in order]


def _rows(shape, gen, outliers, sigma=0.5):
    """N(0, 1) entries times a per-token lognormal magnitude, some channels x8 (K)."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.empty(shape[:-1] + (1,), device="cuda").log_normal_(0.0, sigma, generator=gen)
    if outliers:
        x[..., OUTLIERS] *= 8
    return x


def _pack(codes, bits):
    """Codes [..., n] (n * bits a multiple of 16) -> LSB-first 16-bit halves [..., n * bits / 16] int32."""
    shift = torch.arange(bits, device=codes.device, dtype=torch.uint8)
    stream = ((codes[..., None] >> shift) & 1).reshape(codes.shape[:-1] + (codes.shape[-1] * bits // 16, 16))
    return (stream.to(torch.int32) << torch.arange(16, device=codes.device)).sum(-1, dtype=torch.int32)


def _fields(x, bits, order):
    """Blocks x [n, 64, 128] fp32 -> one half of their records, uint8 [n, code bytes + 768]."""
    n = x.shape[0]
    norm = x.square().sum(-1, keepdim=True).sqrt()
    unit = x / norm.clamp_min(1e-12)
    low, high = unit.amin(1, keepdim=True), unit.amax(1, keepdim=True)
    step = (high - low) / (2 ** bits - 1)
    codes = ((unit - low) / step).round().clamp(0, 2 ** bits - 1).to(torch.uint8)
    low, step, norm = low.half(), step.half(), norm.half()
    back = low.float() + step.float() * codes.float()
    alpha = norm.float() / back.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-12)
    halves = _pack(codes, bits)  # [n, 64, 8 * bits]
    if order == 2:  # each 32-code group as words [half m of its first half | of its second]
        halves = halves.reshape(n, 64, 4, 2, bits).transpose(-1, -2)
    else:  # rows 2j and 2j + 1 interleaved
        halves = halves.reshape(n, 32, 2, 8 * bits).transpose(-1, -2)
    halves = torch.where(halves >= 32768, halves - 65536, halves).to(torch.int16).contiguous()
    raw = [halves.reshape(n, -1).view(torch.uint8), low.reshape(n, -1).view(torch.uint8),
           step.reshape(n, -1).view(torch.uint8), alpha.reshape(n, -1).contiguous().view(torch.uint8)]
    return torch.cat(raw, -1)


def _records(h, pages, bits, gen):
    """Block records [h, pages, 2 * (code bytes + 768)] of K and V drawn like a model's."""
    size = BLOCK * DIM * bits // 8 + 768
    rec = torch.empty((h, pages, 2 * size), dtype=torch.uint8, device="cuda")
    for j in range(h):
        rec[j, :, :size] = _fields(_rows((pages, BLOCK, DIM), gen, True), bits, 2)
        rec[j, :, size:] = _fields(_rows((pages, BLOCK, DIM), gen, False), bits, 1)
    return rec


def prepare(case, seed):
    gen, c = _gen(seed), dict(case)
    return {"prompt": _prepare_prompt, "prefix": _prepare_prefix, "fork": _prepare_fork,
            "compact": _prepare_compact}[c["op"]](c, gen)


def _prepare_prompt(c, gen):
    T, hq, h, dt = c["tokens"], c["hq"], c["h"], DTYPES[c["dtype"]]
    lens = _lengths(c["seqs"], T, c["ragged"], gen)
    cu = torch.tensor([0] + lens, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
    q = torch.randn((T, hq, DIM), generator=gen, device="cuda")
    k, v = _rows((T, h, DIM), gen, True), _rows((T, h, DIM), gen, False)
    if c["fused"]:  # rows of the fused projection: q | k | v
        qkv = torch.cat([q, k, v], 1).to(dt)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + h], qkv[:, hq + h:]
    else:
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    return dict(c, q=q, k=k, v=v, cu=cu, longest=max(lens))


def _prepare_prefix(c, gen):
    hq, h, n, groups, rows, dt = c["hq"], c["h"], c["blocks"], c["groups"], c["rows"], DTYPES[c["dtype"]]
    counts = [n] + [max(1, n * (3 + g) // (4 + 2 * g)) for g in range(1, groups)]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((groups, n), dtype=torch.int32, device="cuda")
    at = 0
    for g, m in enumerate(counts):
        table[g, :m] = order[at:at + m]
        at += m
    split = [0] + _lengths(groups, rows, groups > 1, gen)
    state = dict(c, records=_records(h, pages, c["bits"], gen), table=table,
                 n_pages=torch.tensor(counts, dtype=torch.int32, device="cuda"),
                 row_offsets=torch.tensor(split, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32),
                 row_index=torch.randperm(rows, generator=gen, device="cuda").to(torch.int32),
                 max_rows=max(split),
                 q=torch.randn((rows, hq, DIM), generator=gen, device="cuda").to(dt),
                 # what the rows' own tokens gave: a few hundred of them, none for the first row
                 o_part=torch.randn((rows, hq, DIM), generator=gen, device="cuda") * 0.2,
                 lse_part=torch.randn((rows, hq), generator=gen, device="cuda") + 6.0)
    state["o_part"][0] = 0
    state["lse_part"][0] = -math.inf
    return state


def _spread(n, top, gen):
    """n whole numbers over [0, top], the same set for every seed, in the seed's order."""
    x = torch.arange(n, device="cuda") * top // max(1, n - 1) if n > 1 else torch.tensor([top // 2], device="cuda")
    return x[torch.randperm(n, generator=gen, device="cuda")].to(torch.int32)


def _prepare_fork(c, gen):
    B, MB, h, dt = c["batch"], c["max_blocks"], c["h"], DTYPES[c["dtype"]]
    seqs = torch.randperm(B, generator=gen, device="cuda").to(torch.int32)
    src_of = torch.arange(c["targets"], device="cuda") % c["sources"]
    n_blocks = 1 + _spread(B, MB - 2, gen)
    tail_len = torch.zeros(B, dtype=torch.int32, device="cuda")
    tail_len[seqs[:c["sources"]].long()] = _spread(c["sources"], BLOCK - 1, gen)
    tail_len[seqs[c["sources"]:].long()] = _spread(B - c["sources"], BLOCK - 1, gen)
    # every sequence holds its sealed blocks and one reserved page; page 0 is the pool's unassigned page
    table = 1 + torch.randperm(B * MB, generator=gen, device="cuda").to(torch.int32).reshape(B, MB)
    held = torch.arange(MB, device="cuda")[None] < n_blocks[:, None] + 1
    table = torch.where(held, table, torch.zeros_like(table))
    refs = torch.zeros(B * MB + 1, dtype=torch.int32, device="cuda")
    refs.index_add_(0, table.reshape(-1).long(), (table.reshape(-1) > 0).to(torch.int32))
    refs[0] = 1
    tails = [_rows((B, h, BLOCK, DIM), gen, o).to(dt) for o in (True, False)]
    return dict(c, table=table, n_blocks=n_blocks, tail_len=tail_len, refs=refs, k_tail=tails[0], v_tail=tails[1],
                src=seqs[:c["sources"]][src_of].contiguous(),
                dst=seqs[c["sources"]:c["sources"] + c["targets"]].contiguous())


def _prepare_compact(c, gen):
    P, L, h, B, MB = c["pages"], c["live"], c["h"], c["batch"], c["max_blocks"]
    size = 2 * (BLOCK * DIM * c["bits"] // 8 + 768)
    records = torch.randint(0, 256, (h, P, size), generator=gen, dtype=torch.uint8, device="cuda")
    norms = [torch.rand((h, P, BLOCK), generator=gen, device="cuda").half() for _ in range(2)]
    # page 0 is always live; of the other live pages, `moves` lie at or above index `live`
    low = 1 + torch.randperm(L - 1, generator=gen, device="cuda")[:L - 1 - c["moves"]]
    high = L + torch.randperm(P - L, generator=gen, device="cuda")[:c["moves"]]
    used = torch.cat([low, high])
    used = used[torch.randperm(used.numel(), generator=gen, device="cuda")].to(torch.int32)
    table = torch.zeros(B * MB, dtype=torch.int32, device="cuda")
    table[torch.randperm(B * MB, generator=gen, device="cuda")[:used.numel()]] = used
    table[:MB // 3] = used[:MB // 3] if used.numel() >= MB // 3 else 0  # shared by forks: listed twice
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    refs.index_add_(0, table.long(), (table > 0).to(torch.int32))
    refs[used.long()] = refs[used.long()].clamp_min(1)  # pages held outside the table
    refs[0] = 1
    return dict(c, records=records, k_norm=norms[0], v_norm=norms[1], table=table.reshape(B, MB), refs=refs)


# ------------------------------------------------------------------------------ one pass
def run(state):
    if state["op"] == "prompt":
        out, lse = _prompt_own(state) if own else _prompt_plain(state)
        return {"out": out, "lse": lse}
    if state["op"] == "prefix":
        out, lse = _prefix_own(state) if own else _prefix_plain(state)
        return {"out": out, "lse": lse}
    if state["op"] == "fork":
        (_fork_own if own else _fork_plain)(state)
        return {"table": state["table"], "refs": state["refs"], "n_blocks": state["n_blocks"],
                "tail_len": state["tail_len"], "k_tail": state["k_tail"].view(torch.int16),
                "v_tail": state["v_tail"].view(torch.int16)}
    table, refs, live = _compact_own(state) if own else _compact_plain(state)
    return {"table": table, "refs": refs, "live": live, "records": state["records"],
            "k_norm": state["k_norm"].view(torch.int16), "v_norm": state["v_norm"].view(torch.int16)}


def _prompt_own(s):
    from nsn_b200.prompt import prompt_attention
    return prompt_attention(s["q"], s["k"], s["v"], s["cu"], s["longest"])


def _prefix_own(s):
    from nsn_b200.prefix import prefix_attention
    return prefix_attention(s["q"], s["records"], s["table"], s["n_pages"], bits=s["bits"],
                            row_offsets=s["row_offsets"], row_index=s["row_index"], max_rows=s["max_rows"],
                            o_part=s["o_part"], lse_part=s["lse_part"])


def _fork_own(s):
    from nsn_b200.pages import fork_sequences
    fork_sequences(s["table"], s["n_blocks"], s["tail_len"], s["refs"], s["k_tail"], s["v_tail"], s["src"], s["dst"])


def _compact_own(s):
    from nsn_b200.pages import compact_pages
    return compact_pages([s["records"], s["k_norm"], s["v_norm"]], s["table"], s["refs"])


# --------------------------------------------------------------------------- plain forms
def _prompt_plain(s):
    q, k, v, cu = s["q"].float(), s["k"].float(), s["v"].float(), s["cu"].long()
    T, hq, h = q.shape[0], q.shape[1], k.shape[1]
    lens = cu[1:] - cu[:-1]
    pos = torch.arange(s["longest"], device=q.device)
    at = (cu[:-1, None] + pos).clamp(max=T - 1)  # [seqs, longest]: every sequence padded to the longest
    seqs, n = at.shape
    qp = q[at].reshape(seqs, n, h, hq // h, DIM).permute(0, 2, 3, 1, 4).reshape(seqs, h, hq // h * n, DIM)
    kp, vp = k[at].permute(0, 2, 3, 1), v[at].permute(0, 2, 1, 3)
    x = torch.matmul(qp * SCALE, kp).reshape(seqs, h, hq // h, n, n)
    seen = (pos[None, :] <= pos[:, None])[None] & (pos < lens[:, None])[:, None, :]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.reshape(seqs, h, hq // h * n, n), vp).reshape(seqs, h, hq // h, n, DIM) / total
    lse = (top + total.log())[..., 0]
    real = pos < lens[:, None]
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, n, hq, DIM)[real]
    return out.to(s["q"].dtype), lse.permute(0, 3, 1, 2).reshape(seqs, n, hq)[real]


def _restore_plain(half, bits, order, dtype):
    """One half of gathered records [..., code bytes + 768] -> fp32 rows [..., 64, 128] rounded to dtype."""
    lead, cb = tuple(half.shape[:-1]), BLOCK * DIM * bits // 8
    halves = half[..., :cb].contiguous().view(torch.int16).to(torch.int32) & 0xFFFF
    if order == 2:
        halves = halves.reshape(lead + (64, 4, bits, 2)).transpose(-1, -2)
    else:
        halves = halves.reshape(lead + (32, 8 * bits, 2)).transpose(-1, -2)
    halves = halves.reshape(lead + (64, 4, 2 * bits))
    bit = bits * torch.arange(32, device=half.device)
    first, second = bit // 16, (bit // 16 + 1).clamp(max=2 * bits - 1)
    codes = ((halves[..., first] | (halves[..., second] << 16)) >> (bit % 16)) & (2 ** bits - 1)
    codes = codes.reshape(lead + (64, DIM)).float()
    low = half[..., cb:cb + 256].contiguous().view(torch.float16).float()
    step = half[..., cb + 256:cb + 512].contiguous().view(torch.float16).float()
    alpha = half[..., cb + 512:cb + 768].contiguous().view(torch.float32)
    rows = (low[..., None, :] + step[..., None, :] * codes) * alpha[..., None]
    return rows.to(dtype).float()


def _prefix_plain(s):
    q, rec, dt = s["q"], s["records"], s["q"].dtype
    rows, hq, h, groups = q.shape[0], s["hq"], s["h"], s["groups"]
    half, n = rec.shape[-1] // 2, s["table"].shape[1]
    got = rec[:, s["table"].long()].transpose(0, 1)  # [groups, h, blocks, record]
    k = _restore_plain(got[..., :half], s["bits"], 2, dt).reshape(groups, h, n * BLOCK, DIM)
    v = _restore_plain(got[..., half:], s["bits"], 1, dt).reshape(groups, h, n * BLOCK, DIM)
    off = s["row_offsets"].long()
    pos = torch.arange(s["max_rows"], device=q.device)
    at = s["row_index"].long()[(off[:-1, None] + pos).clamp(max=rows - 1)]  # [groups, max_rows]
    qp = q.float()[at].reshape(groups, s["max_rows"], h, hq // h, DIM).permute(0, 2, 1, 3, 4)
    qp = qp.reshape(groups, h, s["max_rows"] * (hq // h), DIM)
    x = torch.matmul(qp * SCALE, k.transpose(-1, -2))
    seen = torch.arange(n * BLOCK, device=q.device) < BLOCK * s["n_pages"].long()[:, None]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, v) / total
    lse = (top + total.log())[..., 0]
    real = pos < (off[1:] - off[:-1])[:, None]
    o = o.reshape(groups, h, s["max_rows"], hq // h, DIM).transpose(1, 2).reshape(groups, s["max_rows"], hq, DIM)
    lse = lse.reshape(groups, h, s["max_rows"], hq // h).transpose(1, 2).reshape(groups, s["max_rows"], hq)
    order = at[real]
    o, lse = torch.empty_like(s["o_part"]).index_copy(0, order, o[real]), \
        torch.empty_like(s["lse_part"]).index_copy(0, order, lse[real])
    top = torch.maximum(lse, s["lse_part"])
    a, b = (lse - top).exp(), (s["lse_part"] - top).exp()
    out = (o * a[..., None] + s["o_part"] * b[..., None]) / (a + b)[..., None]
    return out.to(dt), top + (a + b).log()


def _fork_plain(s):
    table, n_blocks, tail_len, refs, src, dst = (s["table"], s["n_blocks"], s["tail_len"], s["refs"], s["src"].long(),
                                                 s["dst"].long())
    old = table[dst].reshape(-1)
    refs.index_add_(0, old.long(), -(old > 0).to(torch.int32))
    sealed = torch.arange(table.shape[1], device=table.device) < n_blocks[src][:, None]
    new = torch.where(sealed, table[src], torch.zeros_like(table[src]))
    refs.index_add_(0, new.reshape(-1).long(), (new.reshape(-1) > 0).to(torch.int32))
    table[dst] = new
    n_blocks[dst] = n_blocks[src]
    tail_len[dst] = tail_len[src]
    used = (torch.arange(BLOCK, device=table.device) < tail_len[src][:, None])[:, None, :, None]
    s["k_tail"][dst] = torch.where(used, s["k_tail"][src], s["k_tail"][dst])
    s["v_tail"][dst] = torch.where(used, s["v_tail"][src], s["v_tail"][dst])


def _compact_plain(s):
    refs, table = s["refs"], s["table"]
    used = refs > 0
    live = used.sum(dtype=torch.int32).reshape(1)
    page = torch.arange(refs.numel(), device=refs.device)
    src, dst = page[used & (page >= live)], page[~used & (page < live)]
    to = page.to(torch.int32).index_copy(0, src, dst.to(torch.int32))
    s["records"][:, dst] = s["records"][:, src]
    s["k_norm"][:, dst] = s["k_norm"][:, src]
    s["v_norm"][:, dst] = s["v_norm"][:, src]
    packed = torch.zeros_like(refs).index_copy(0, to[used].long(), refs[used])
    return to[table.long()], packed, live


# ---------------------------------------------------------------------- 64-bit definition
def exact(case, seed):
    if case["op"] == "prompt":
        return _prompt_exact(prepare(case, seed))
    if case["op"] == "prefix":
        return _prefix_exact(prepare(case, seed))
    return None  # copies and whole numbers


def _attend64(q, k, v, first=None):
    """Rows q over keys k, values v; with ``first``, row i sees the keys up to first + i."""
    w = torch.einsum("id,jd->ij", q, k) / math.sqrt(DIM)
    if first is not None:
        i, j = torch.arange(q.shape[0], device=q.device), torch.arange(k.shape[0], device=q.device)
        w = torch.where(j[None, :] - i[:, None] > first, torch.full_like(w, -math.inf), w)
    lse = torch.logsumexp(w, 1)
    return torch.einsum("ij,jd->id", torch.exp(w - lse[:, None]), v), lse


def _prompt_exact(s):
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    ends = s["cu"].tolist()
    for a, b in zip(ends[:-1], ends[1:]):
        for j in range(q.shape[1]):
            kv = j // (q.shape[1] // k.shape[1])
            for i in range(a, b, 4096):
                e = min(b, i + 4096)
                out[i:e, j], lse[i:e, j] = _attend64(q[i:e, j], k[a:e, kv], v[a:e, kv], i - a)
    return {"out": out, "lse": lse}


def _codes64(raw, bits):
    """Bytes [n, rows, 16 * bits] of LSB-first streams -> whole numbers [n, rows, 128]."""
    stream = (raw[..., None].long() >> torch.arange(8, device=raw.device)) & 1
    stream = stream.reshape(raw.shape[:-1] + (DIM, bits))
    return (stream << torch.arange(bits, device=raw.device)).sum(-1)


def _blocks64(half, bits, rows_paired, dtype):
    cb = BLOCK * DIM * bits // 8
    n = half.shape[0]
    two = half[:, :cb].reshape(n, -1, 2, 2)  # 32-bit words as two 16-bit halves of two bytes
    if rows_paired:
        raw = two.reshape(n, 32, 8 * bits, 2, 2).permute(0, 1, 3, 2, 4)
    else:
        raw = two.reshape(n, 64, 4, bits, 2, 2).permute(0, 1, 2, 4, 3, 5)
    codes = _codes64(raw.reshape(n, BLOCK, 16 * bits), bits).double()
    low = half[:, cb:cb + 256].contiguous().view(torch.float16).double()[:, None]
    step = half[:, cb + 256:cb + 512].contiguous().view(torch.float16).double()[:, None]
    alpha = half[:, cb + 512:].contiguous().view(torch.float32).double()[:, :, None]
    return ((low + step * codes) * alpha).to(dtype).double().reshape(n * BLOCK, DIM)


def _prefix_exact(s):
    q, rec, dt = s["q"].double(), s["records"], s["q"].dtype
    G, half = s["hq"] // s["h"], rec.shape[-1] // 2
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    ends, counts = s["row_offsets"].tolist(), s["n_pages"].tolist()
    for g, m in enumerate(counts):
        rows = s["row_index"][ends[g]:ends[g + 1]].long()
        for j in range(s["h"]):
            blocks = rec[j, s["table"][g, :m].long()]
            k = _blocks64(blocks[:, :half], s["bits"], False, dt)
            v = _blocks64(blocks[:, half:], s["bits"], True, dt)
            for i in range(j * G, j * G + G):
                o, e = _attend64(q[rows, i], k, v)
                both = torch.logaddexp(e, s["lse_part"][rows, i].double())
                out[rows, i] = o * torch.exp(e - both)[:, None] + s["o_part"][rows, i].double() * torch.exp(
                    s["lse_part"][rows, i].double() - both)[:, None]
                lse[rows, i] = both
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "prompt":
        T, hq, h = c["tokens"], c["hq"], c["h"]
        lens = _work_lengths(c["seqs"], T, c["ragged"])
        pairs = sum(n * (n + 1) / 2 for n in lens)
        return {"bytes": 2.0 * T * DIM * (2 * hq + 2 * h) + 4.0 * T * hq, "flops": 4.0 * DIM * hq * pairs}
    if c["op"] == "prefix":
        n, groups, rows, hq, h = c["blocks"], c["groups"], c["rows"], c["hq"], c["h"]
        counts = [n] + [max(1, n * (3 + g) // (4 + 2 * g)) for g in range(1, groups)]
        size = 2 * (BLOCK * DIM * c["bits"] // 8 + 768)
        per = sorted(_work_lengths(groups, rows, groups > 1))  # the seed deals them out: their mean
        pairs = sum(counts) / groups * BLOCK * sum(per)
        moved = rows * hq * (DIM * (2 + 2 + 4) + 8.0)  # q, out, o_part, both log-sum-exps
        return {"bytes": h * size * float(sum(counts)) + moved, "flops": 4.0 * DIM * hq * pairs}
    if c["op"] == "fork":
        row = c["h"] * DIM * 2 * 2.0
        mean = (BLOCK - 1) / 2
        sources, targets = min(c["sources"], c["targets"]), c["targets"]
        ints = 4.0 * c["max_blocks"] * (sources + 2 * targets) + 4.0 * c["max_blocks"] * targets
        return {"bytes": row * mean * (sources + targets) + ints, "flops": 0.0}
    size = 2 * (BLOCK * DIM * c["bits"] // 8 + 768) + 2 * BLOCK * 2
    ints = 4.0 * (2 * c["pages"] + 2 * c["batch"] * c["max_blocks"])
    return {"bytes": 2.0 * c["moves"] * c["h"] * size + ints, "flops": 0.0}


def _work_lengths(n, total, ragged):
    """The lengths of ``_lengths`` without their order."""
    if n == 1:
        return [total]
    if not ragged:
        return [total // n + (1 if i < total % n else 0) for i in range(n)]
    weight = [math.exp(3.0 * i / (n - 1)) for i in range(n)]
    got = [1 + int((total - n) * w / sum(weight)) for w in weight]
    got[-1] += total - sum(got)
    got[0], got[-1] = 1, got[-1] + got[0] - 1
    return got
