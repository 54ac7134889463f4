"""Shared-prefix attention against its definition in 64 bits over real block records: code
widths, types, groups, row orders, merges, empty prefixes, statuses and refusals."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def pool(h, pages, bits, seed=0):
    """Block records of `pages` pages encoded by the library from K / V rows of a model's kind."""
    from nsn_b200 import paged, primitives as w
    g = torch.Generator(device="cuda").manual_seed(seed)
    rec, kp, vp = paged.block_record_pools(h, pages, bits, "cuda")
    for p, boost in ((kp, True), (vp, False)):
        x = torch.randn((h, pages, 64, 128), generator=g, device="cuda") * torch.exp(
            0.5 * torch.randn((h, pages, 64, 1), generator=g, device="cuda"))
        if boost:
            x[..., [3, 37, 71, 105]] *= 8
        w.encode_blocks(x.half(), bits, out=p, out_row_stride=pages, out_offset=0, check=False)
    return rec, kp, vp


def rows_of(p, bits, dtype):
    """Restored rows [h, pages, 64, 128] in dtype: alpha * (min + scale * code), rounded in fp32."""
    from nsn_b200 import primitives as w
    h, pages = p["codes"].shape[:2]
    raw = w.from_code_order(p["codes"].contiguous(), bits, p["code_order"]).reshape(h, pages, -1)
    stream = ((raw[..., None].int() >> torch.arange(8, device="cuda")) & 1).reshape(h, pages, 64, 128, bits)
    codes = (stream << torch.arange(bits, device="cuda")).sum(-1).double()
    d = (p["min"].double()[:, :, None] + p["scale"].double()[:, :, None] * codes).float()
    return (d * p["alpha"][..., None]).to(dtype)


def reference(q, k, v, table, counts, offsets, index, o_part, lse_part):
    """out, lse and their error bounds (see tests/test_gpu_prompt.py) in 64 bits."""
    rows, hq = q.shape[:2]
    h, u = k.shape[0], U[q.dtype]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64, device="cuda")
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    groups = {r: g for g in range(len(counts)) for r in index[offsets[g]:offsets[g + 1]]}
    for r in range(rows):
        pages = table[groups[r]][:counts[groups[r]]] if r in groups else []
        n = 64 * len(pages)
        for j in range(hq):
            kv = j // (hq // h)
            kk = k[kv, pages].reshape(n, 128).double() if n else torch.zeros((0, 128), device="cuda").double()
            vv = v[kv, pages].reshape(n, 128).double() if n else kk
            x = kk @ q[r, j].double() / math.sqrt(128)
            dx = 2.0 ** -20 * (1 + float((kk.abs() @ q[r, j].double().abs()).max() / math.sqrt(128) if n else 0))
            rest = o_part[r, j].double() if o_part is not None else torch.zeros(128, device="cuda").double()
            e = lse_part[r, j].double() if lse_part is not None else torch.tensor(-math.inf, device="cuda").double()
            both = torch.logaddexp(torch.logsumexp(x, 0), e) if n else e
            if both == -math.inf:
                continue
            p, b = torch.exp(x - both), torch.exp(e - both)
            o, big = p @ vv + b * rest, p @ vv.abs() + b * rest.abs()
            out[r, j], lse[r, j] = o, both
            tol[r, j] = u * (o.abs() + big) * 1.01 + (2 * dx + 2.0 ** -20) * big
            if n:
                tol[r, j] += n * 2.0 ** -25 * vv.abs().amax()
            ltol[r, j] = dx + 2.0 ** -21 * (both.abs() + 1)
    return out, lse, tol, ltol


def check(got, ref):
    (out, lse), (o, e, tol, ltol) = got, ref
    d = (out.double() - o).abs()
    assert bool((d <= tol).all()), f"out off by {float((d - tol).max())} over its bound"
    same = (lse.double() == e) | ((lse.double() - e).abs() <= ltol)
    assert bool(same.all()), f"lse off by {float((lse.double() - e).abs().nan_to_num().max())}"


def case(h, G, bits, dtype, counts, per_group, seed=0, part=True, spare=2, loose=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    pages = sum(counts) + spare
    rec, kp, vp = pool(h, pages, bits, seed)
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table, at = [], 0
    for n in counts:
        table.append(order[at:at + n])
        at += n
    rows = sum(per_group) + loose
    index = torch.randperm(rows, generator=g, device="cuda").tolist()
    offsets = [sum(per_group[:i]) for i in range(len(per_group) + 1)]
    hq = h * G
    q = torch.randn((rows, hq, 128), generator=g, device="cuda").to(dtype)
    o_part = lse_part = None
    if part:
        o_part = torch.randn((rows, hq, 128), generator=g, device="cuda")
        lse_part = 5 + torch.randn((rows, hq), generator=g, device="cuda")
        o_part[0], lse_part[0] = 0, -math.inf
    wide = max(counts + [1])
    t = torch.tensor([r + [0] * (wide - len(r)) for r in table], dtype=torch.int32, device="cuda").reshape(-1, wide)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    args = dict(bits=bits, row_offsets=dev(offsets), row_index=dev(index), max_rows=max(per_group), o_part=o_part,
                lse_part=lse_part)
    ref = reference(q, rows_of(kp, bits, dtype), rows_of(vp, bits, dtype), table, counts, offsets, index, o_part,
                    lse_part)
    return (q, rec, t, dev(counts)), args, ref


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [3, 5])
@pytest.mark.parametrize("h,G,counts,per_group", [
    (2, 4, [1], [1]), (1, 1, [3], [1]), (2, 2, [5], [70]), (3, 3, [2], [17]), (2, 8, [9], [9]), (1, 4, [33], [40]),
    (2, 4, [4, 1, 7], [3, 9, 1]), (2, 4, [0, 3], [4, 4]), (1, 6, [2, 2], [1, 60]), (8, 4, [20], [2]),
    (2, 1, [130], [2]), (1, 16, [6], [20]), (1, 4, [5], [300]), (1, 8, [3, 6], [150, 200]), (2, 6, [7, 0], [260, 9])])
def test_groups_and_lengths(h, G, counts, per_group, bits, dtype):
    from nsn_b200.prefix import prefix_attention
    a, kw, ref = case(h, G, bits, dtype, counts, per_group)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(prefix_attention(*a, status=status, **kw), ref)
    assert int(status) == 0


@pytest.mark.parametrize("rows", [31, 32, 33, 63, 64, 65, 127, 129, 200])
def test_row_tiles(rows):
    """Row counts around the kernels' tile sizes."""
    from nsn_b200.prefix import prefix_attention
    a, kw, ref = case(1, 4, 3, torch.float16, [3], [rows], seed=rows)
    check(prefix_attention(*a, **kw), ref)


@pytest.mark.parametrize("bits,counts,rows", [(3, [3], [300]), (5, [4, 5], [70, 200]), (3, [1], [97])])
def test_max_rows_only_sizes_the_launch(bits, counts, rows):
    """Fewer row tiles launched than the groups have: a CTA takes several in turn."""
    from nsn_b200.prefix import prefix_attention
    a, kw, ref = case(1, 4, bits, torch.float16, counts, rows, seed=9)
    kw["max_rows"] = 1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(prefix_attention(*a, status=status, **kw), ref)
    assert int(status) == 0


def test_rows_outside_every_group_and_no_partial():
    from nsn_b200.prefix import prefix_attention
    a, kw, ref = case(2, 4, 3, torch.float16, [3, 2], [2, 3], loose=4)
    check(prefix_attention(*a, **kw), ref)
    a, kw, ref = case(2, 4, 3, torch.float16, [0, 2], [2, 3], part=False, loose=2)
    out, lse = prefix_attention(*a, **kw)
    check((out, lse), ref)
    assert bool((lse == -math.inf).sum() == 4 * 8) and bool((out[lse == -math.inf] == 0).all())


def test_plain_arguments_are_one_group_in_order():
    from nsn_b200.prefix import prefix_attention
    (q, rec, t, n), kw, _ = case(2, 4, 3, torch.float16, [6], [10], part=False)
    kw["row_index"] = None
    a = prefix_attention(q, rec, t, n, **kw)
    b = prefix_attention(q, rec, t[0], bits=3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_strided_records_and_wider_table():
    """A pool inside a larger one, and a table with more columns than pages in use."""
    from nsn_b200.prefix import prefix_attention
    (q, rec, t, n), kw, ref = case(2, 2, 3, torch.float16, [4], [5])
    big = torch.zeros((3, rec.shape[1] + 9, rec.shape[2] + 256), dtype=torch.uint8, device="cuda")
    big[:2, 4:4 + rec.shape[1], :rec.shape[2]] = rec
    wide = torch.full((1, 50), 10 ** 9, dtype=torch.int32, device="cuda")
    wide[:, :4] = t
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(prefix_attention(q, big[:2, 4:4 + rec.shape[1], :rec.shape[2]], wide, n, status=status, **kw), ref)
    assert int(status) == 0


@pytest.mark.parametrize("bits", [3, 5])
def test_agrees_with_the_bridge_rounding_cache(bits):
    """One sequence, whole context in the prefix: the paged cache's restore-kernel attention."""
    from nsn_b200.paged import PagedKVCache
    from nsn_b200.prefix import prefix_attention
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn((2, 64 * 7, 128), generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn((1, 8, 128), generator=g, device="cuda").half()
    kv = PagedKVCache(1, 2, 8, bits=bits, hq=8, restore_rounding="kv")
    rec = PagedKVCache(1, 2, 8, bits=bits, hq=8)
    for c in (kv, rec):
        c.prefill(0, k, v)
    want = kv.attend(q).double()
    out, _ = prefix_attention(q, rec.records, rec.block_table[:, :7], bits=bits)
    # both round K, V, p-free: two fp16 roundings of the output plus p's rounding here
    assert float((out.double() - want).abs().max()) <= 3 * 2.0 ** -11 * float(want.abs().max()) + 2.0 ** -11


def test_statuses():
    from nsn_b200.prefix import prefix_attention
    for what, bit in (("page", 128), ("meta", 1), ("q", 1)):
        (q, rec, t, n), kw, _ = case(1, 2, 3, torch.float16, [3], [4])
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        if what == "page":
            t[0, 1] = rec.shape[1]
        if what == "meta":
            at = rec.shape[2] // 2 - 768  # behind K's codes: the channels' minima
            rec[0, int(t[0, 2]), at:at + 2] = 255  # NaN
        if what == "q":
            q[1, 0, 5] = math.inf
        prefix_attention(q, rec, t, n, status=status, **kw)
        assert int(status) & bit


def test_same_result_twice_on_streams_and_in_a_graph():
    from nsn_b200.prefix import prefix_attention
    a, kw, ref = case(2, 4, 3, torch.bfloat16, [40], [33])
    one = prefix_attention(*a, **kw)
    check(one, ref)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        two = prefix_attention(*a, **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        prefix_attention(*a, out=one[0], lse=one[1], **kw)
    one[0].zero_()
    graph.replay()
    assert torch.equal(one[0], two[0])


def test_refusals():
    from nsn_b200 import ContractError
    from nsn_b200._lib import NativeError
    from nsn_b200.prefix import prefix_attention
    (q, rec, t, n), kw, _ = case(2, 2, 3, torch.float16, [2], [3])
    bads = [dict(q=q.float()), dict(q=q[:, :3].contiguous()), dict(rec=rec[..., :-16]), dict(t=t.long()),
            dict(n=n.long()), dict(bits=4), dict(bits=5), dict(row_index=kw["row_index"][:2]),
            dict(row_offsets=kw["row_offsets"][:1]), dict(lse_part=None), dict(o_part=kw["o_part"].half()),
            dict(q=q.cpu()), dict(t=torch.cat([t, t]), row_offsets=None)]
    for bad in bads:
        a = dict(q=q, rec=rec, t=t, n=n) | {k: x for k, x in bad.items() if k in ("q", "rec", "t", "n")}
        b = kw | {k: x for k, x in bad.items() if k not in ("q", "rec", "t", "n")}
        with pytest.raises(ContractError):
            prefix_attention(a["q"], a["rec"], a["t"], a["n"], **b)
    with pytest.raises(NativeError):
        prefix_attention(q, rec, t, n, ws=torch.empty(16, dtype=torch.uint8, device="cuda"), **kw)


def test_a_graph_keeps_its_workspace():
    """Warmed up and captured on one stream, a larger eager call there afterwards, and new tensors
    where its old buffer was: a replay gives what the call gave and writes nothing else."""
    from nsn_b200.prefix import prefix_attention
    a, kw, ref = case(2, 4, 3, torch.float16, [40], [33])
    b, kb, big = case(2, 4, 3, torch.float16, [30], [300], seed=2)
    out, lse = torch.empty_like(a[0]), torch.empty((33, 8), device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        prefix_attention(*a, out=out, lse=lse, **kw)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        prefix_attention(*a, out=out, lse=lse, **kw)
    with torch.cuda.stream(s):
        check(prefix_attention(*b, **kb), big)
        others = [torch.full((1 << 18,), 7.0, device="cuda") for _ in range(64)]
        out.zero_()
        graph.replay()
    s.synchronize()
    check((out, lse), ref)
    assert all(bool((x == 7).all()) for x in others)
    with torch.cuda.stream(s):  # eager calls there while the graph replays elsewhere
        got = [prefix_attention(*b, **kb) for _ in range(20)]
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    check((out, lse), ref)
    for x in got:
        check(x, big)


def test_threads_on_one_stream():
    """Two host threads enqueue on the same stream; each call joins its own chunks."""
    import threading
    from nsn_b200.prefix import prefix_attention
    cases = [case(2, 4, 3, torch.float16, [40], [33], seed=s) for s in (1, 2)]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        a, kw, _ = cases[i]
        got[i] += [prefix_attention(*a, **kw) for _ in range(200)]
    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in (0, 1):
        check(got[i][0], cases[i][2])
        assert all(torch.equal(o, got[i][0][0]) and torch.equal(e, got[i][0][1]) for o, e in got[i])


@pytest.mark.parametrize("blocks,rows,part", [(1, 3, True), (1, 3, False), (40, 3, True), (2, 70, True), (0, 3, True)])
def test_a_row_without_a_finite_score_is_nan(blocks, rows, part):
    """A NaN query's output and log-sum-exp are NaN over any prefix, with its own finite part or
    without; the other rows keep theirs."""
    from nsn_b200.prefix import prefix_attention
    a, kw, ref = case(1, 4, 3, torch.float16, [blocks], [rows], part=part)
    a[0][1] = math.nan
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = prefix_attention(*a, status=status, **kw)
    if blocks:
        assert bool(out[1].isnan().all()) and bool(lse[1].isnan().all()) and int(status) & 1
    keep = torch.arange(rows, device="cuda") != 1 if blocks else slice(None)  # no prefix: q is not read
    check((out[keep], lse[keep]), [t[keep] for t in ref])


@pytest.mark.parametrize("blocks", [0, 3])
def test_a_nan_part_is_not_dropped(blocks):
    """A row whose own part has a NaN log-sum-exp is NaN: NaN does not mean "no own tokens"."""
    from nsn_b200.prefix import prefix_attention
    a, kw, ref = case(1, 4, 3, torch.float16, [blocks], [5])
    kw["o_part"][2], kw["lse_part"][2] = math.nan, math.nan
    kw["lse_part"][3] = math.nan  # its output finite
    out, lse = prefix_attention(*a, **kw)
    assert bool(out[2:4].isnan().all()) and bool(lse[2:4].isnan().all())
    keep = torch.tensor([0, 1, 4], device="cuda")
    check((out[keep], lse[keep]), [t[keep] for t in ref])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [3, 5])
def test_rows_are_restored_bit_for_bit(bits, dtype):
    """K and V rows equal alpha (min + scale code), each step rounded to fp32 and the result to
    dtype, for channels whose minimum is small beside their scale (one-signed channels) too.

    Page t holds random codes and a K factor in token t only, so that a row of group t with a
    large q sees that token alone.  Channel 0 of K is the factor itself: with q = 8 along it the
    score is some 1000, p is 1 within 2^-13 and the output the token's V row.  With q along
    channel c the log-sum-exp is q K[c] / sqrt(128) within 2^-21 of its size, which names K[c]
    among the values of dtype (2^-11 apart and more)."""
    from nsn_b200 import paged
    from nsn_b200.prefix import prefix_attention
    g = torch.Generator(device="cuda").manual_seed(bits)
    rec, kp, vp = paged.block_record_pools(1, 64, bits, "cuda")
    mins = torch.tensor([1.0, 0.1, 1e-3, 6e-8, 3e-2, 0.02, 1e-4, 5e-3], device="cuda").repeat(16)
    steps = torch.tensor([0.1, 0.0123, 0.777, 0.05, 0.1, 0.3], device="cuda").repeat(22)[:128]
    for p in (kp, vp):
        p["codes"].copy_(torch.randint(0, 256, p["codes"].shape, generator=g, dtype=torch.uint8, device="cuda"))
        p["min"].copy_(mins.half())
        p["scale"].copy_(steps.half())
    vp["min"][..., 1::3] *= -1
    kp["scale"][..., 0] = 0
    t, c = torch.arange(64, device="cuda"), torch.arange(128, device="cuda")
    kp["alpha"].zero_()
    kp["alpha"][0, t, t] = 1024 * (1 + torch.rand(64, generator=g, device="cuda"))
    vp["alpha"].copy_(torch.rand(vp["alpha"].shape, generator=g, device="cuda") * 20 + 0.1)
    k, v = rows_of(kp, bits, dtype)[0, t, t], rows_of(vp, bits, dtype)[0, t, t]  # [64, 128]
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    size = torch.where(c == 0, 8.0, 32768.0)
    q = torch.diag(size).to(dtype).repeat(64, 1)[:, None].contiguous()  # row 128 t + c: along channel c
    out, lse = prefix_attention(q, rec, dev(list(range(64)))[:, None], dev([1] * 64), bits=bits,
                                row_offsets=dev([128 * i for i in range(65)]), max_rows=128)
    out, lse = out.reshape(64, 128, 128), lse.reshape(64, 128)
    assert torch.equal(out[:, 0], v)
    known = k.float() * size / math.sqrt(128) > 150  # the other 63 tokens' p are 0
    assert float(known.float().mean()) > 0.9
    assert torch.equal((lse.double() * math.sqrt(128) / size).to(dtype)[known], k[known])


def test_status_elsewhere_is_refused():
    from nsn_b200 import ContractError
    from nsn_b200.prefix import prefix_attention
    a, kw, _ = case(1, 2, 3, torch.float16, [2], [3])
    for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64, device="cuda")):
        with pytest.raises(ContractError):
            prefix_attention(*a, status=bad, **kw)


def test_workspace_elsewhere_is_refused():
    from nsn_b200 import ContractError
    from nsn_b200.prefix import prefix_attention
    a, kw, _ = case(1, 2, 3, torch.float16, [2], [3])
    big = torch.empty(1 << 20, dtype=torch.uint8)
    for bad in (big, big.cuda()[::2]):
        with pytest.raises(ContractError):
            prefix_attention(*a, ws=bad, **kw)


@pytest.mark.parametrize("growth", ["level", "rising", "spike", "falling"])
@pytest.mark.parametrize("bits,dtype,counts,rows,wide,most", [
    (3, torch.float16, [11], [3], 888, None),          # one row tile, both teams on it: three blocks each
    (5, torch.float16, [13], [3], 888, None),
    (3, torch.bfloat16, [11], [40], 888, None),        # two row tiles, the second in part
    (3, torch.float16, [9, 14], [20, 70], 888, None),
    (5, torch.bfloat16, [17], [300], 180, 1),          # a CTA takes several pairs of row tiles in turn
    (3, torch.float16, [17], [300], 180, 1)])
def test_many_blocks_per_cta(bits, dtype, counts, rows, wide, most, growth):
    """Chunks of several blocks: P.V accumulated, both S buffers used again, the maximum in use
    raised with O rescaled (K of later blocks larger), or never raised."""
    from nsn_b200 import _lib as L
    from nsn_b200.prefix import prefix_attention
    g = torch.Generator(device="cuda").manual_seed(7)
    pages, G = sum(counts) + 2, 4
    rec, kp, vp = pool(1, pages, bits, 5)
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table, at = [], 0
    for n in counts:
        for i, p in enumerate(order[at:at + n]):
            kp["alpha"][:, p] *= {"level": 1.0, "rising": 1.7 ** (i % 6), "spike": 12.0 if i % 6 == 3 else 1.0,
                                  "falling": 1.7 ** (5 - i % 6)}[growth]
        table.append(order[at:at + n])
        at += n
    total = sum(rows)
    q = torch.randn((total, G, 128), generator=g, device="cuda").to(dtype)
    o_part = torch.randn((total, G, 128), generator=g, device="cuda")
    lse_part = 5 + torch.randn((total, G), generator=g, device="cuda")
    index = torch.randperm(total, generator=g, device="cuda").tolist()
    offsets = [sum(rows[:i]) for i in range(len(rows) + 1)]
    t = torch.zeros((len(counts), wide), dtype=torch.int32, device="cuda")
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for i, r in enumerate(table):
        t[i, :len(r)] = dev(r)
    chunks = L.load().nsnkv_prefix_attn_workspace_bytes(total, len(counts), G, 1, wide) // (total * G * 129 * 4)
    assert -(-wide // chunks) >= 4  # blocks per CTA
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = prefix_attention(q, rec, t, dev(counts), bits=bits, row_offsets=dev(offsets), row_index=dev(index),
                           max_rows=most or max(rows), o_part=o_part, lse_part=lse_part, status=status)
    check(got, reference(q, rows_of(kp, bits, dtype), rows_of(vp, bits, dtype), table, counts, offsets, index, o_part,
                         lse_part))
    assert int(status) == 0
