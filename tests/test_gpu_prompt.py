"""Prompt attention against its definition in 64 bits: lengths, types, groups, strides, values
that a row must not see, and refusals."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a unit in the last place, relative


def make(lens, hq, h, dtype, seed=0, fused=False, extra=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lens) + extra
    q = torch.randn((T, hq, 128), generator=g, device="cuda")
    k = torch.randn((T, h, 128), generator=g, device="cuda")
    k[..., [3, 37, 71, 105]] *= 8
    v = torch.randn((T, h, 128), generator=g, device="cuda") * torch.exp(
        0.5 * torch.randn((T, 1, 1), generator=g, device="cuda"))
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    if fused:
        qkv = torch.cat([q, k, v], 1).to(dtype)
        return qkv[:, :hq], qkv[:, hq:hq + h], qkv[:, hq + h:], cu
    return q.to(dtype), k.to(dtype), v.to(dtype), cu


def reference(q, k, v, lens, causal=True):
    """out, lse and an elementwise error bound of out, of lse; all in 64 bits.

    The bound: the output's rounding, u |out|; the probabilities' rounding, u sum p |v| (and
    2^-25 per token where they are subnormal in fp16); the scores' error in fp32 accumulation
    and exponentials, |dx| <= 2^-20 sum |q k| / sqrt(128) + 2^-20 (about 8 of the 128 partial
    sums' units), which moves each p, so the output by 2 |dx| sum p |v| and the lse by |dx|.
    """
    u = U[q.dtype]
    q, k, v = q.double(), k.double(), v.double()
    hq, h = q.shape[1], k.shape[1]
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    tol, ltol = torch.zeros_like(q), torch.zeros_like(lse)
    a = 0
    for n in [n for n in lens if n]:
        for j in range(hq):
            qq, kk, vv = q[a:a + n, j], k[a:a + n, j // (hq // h)], v[a:a + n, j // (hq // h)]
            x = qq @ kk.T / math.sqrt(128)
            dx = 2.0 ** -20 * (1 + (qq.abs() @ kk.abs().T).amax(1) / math.sqrt(128))
            if causal:
                x = x.masked_fill(torch.ones(n, n, device=q.device).triu(1).bool(), -math.inf)
            p = torch.softmax(x, 1)
            o, big = p @ vv, p @ vv.abs()
            out[a:a + n, j], lse[a:a + n, j] = o, torch.logsumexp(x, 1)
            tol[a:a + n, j] = u * (o.abs() + big) * 1.01 + 2 * dx[:, None] * big + n * 2.0 ** -25 * vv.abs().amax()
            ltol[a:a + n, j] = dx + 2.0 ** -22 * lse[a:a + n, j].abs()
        a += n
    return out, lse, tol, ltol


def check(out, lse, ref, rows=slice(None)):
    o, e, tol, ltol = (t[rows] for t in ref)
    d = (out[rows].double() - o).abs()
    assert bool((d <= tol).all()), f"out off by {float((d - tol).max())} over its bound"
    d = (lse[rows].double() - e).abs()
    assert bool((d <= ltol).all()), f"lse off by {float((d - ltol).max())} over its bound"


LENS = [[1], [2], [63], [64], [65], [127], [128], [129], [255], [256], [257], [3, 0, 130, 1, 64, 511], [1] * 37,
        [1500], [700, 1, 900],
        [66] * 140]  # more sequences than the longest-first order keeps in registers


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_lengths(lens, dtype):
    from nsn_b200.prompt import prompt_attention
    q, k, v, cu = make(lens, 8, 2, dtype, seed=len(lens) + lens[0])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = prompt_attention(q, k, v, cu, max(lens), status=status)
    check(out, lse, reference(q, k, v, lens))
    assert int(status) == 0


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("hq,h", [(1, 1), (4, 4), (6, 2), (8, 1), (32, 8), (48, 8), (16, 16), (5, 5)])
def test_heads_and_strides(hq, h, fused):
    from nsn_b200.prompt import prompt_attention
    lens = [70, 333]
    q, k, v, cu = make(lens, hq, h, torch.bfloat16 if fused else torch.float16, fused=fused)
    out, lse = prompt_attention(q, k, v, cu, 333)
    check(out, lse, reference(q, k, v, lens))


@pytest.mark.parametrize("lens", [[1], [200], [129, 600]], ids=str)
def test_not_causal(lens):
    from nsn_b200.prompt import prompt_attention
    q, k, v, cu = make(lens, 4, 2, torch.float16)
    out, lse = prompt_attention(q, k, v, cu, max(lens), causal=False)
    check(out, lse, reference(q, k, v, lens, causal=False))


def test_head_major_strides():
    """Operands laid out [heads, T, 128], as a model's transposed projections are."""
    from nsn_b200.prompt import prompt_attention
    lens = [300, 45]
    q, k, v, cu = make(lens, 8, 4, torch.float16)
    q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    out, lse = prompt_attention(q, k, v, cu, 300)
    check(out, lse, reference(q, k, v, lens))


@pytest.mark.parametrize("lens", [[40], [300, 45]], ids=str)
def test_broadcast_heads_and_unaligned_output(lens):
    """K and V of one head expanded to four (stride 0), and an output that is only 16-byte aligned."""
    from nsn_b200.prompt import prompt_attention
    q, k, v, cu = make(lens, 4, 1, torch.float16)
    ref = reference(q, k, v, lens)
    T = sum(lens)
    wide = prompt_attention(q, k.expand(T, 4, 128), v.expand(T, 4, 128), cu, max(lens))
    check(*wide, ref)
    out = torch.empty(T * 512 + 8, dtype=torch.float16, device="cuda")[8:].view(T, 4, 128)
    prompt_attention(q, k, v, cu, max(lens), out=out)
    check(out, wide[1], ref)


@pytest.mark.parametrize("longest", [1, 64, 100000])
def test_longest_only_sizes_the_launch(longest):
    from nsn_b200.prompt import prompt_attention
    lens = [513, 20]
    q, k, v, cu = make(lens, 4, 2, torch.float16)
    out, lse = prompt_attention(q, k, v, cu, longest)
    check(out, lse, reference(q, k, v, lens))


@pytest.mark.parametrize("lens", [[40, 50], [700, 900]], ids=str)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_unseen_values_do_not_reach_a_row(lens, value):
    """Non-finite K and V of later tokens and of other sequences stay out of the earlier rows."""
    from nsn_b200.prompt import prompt_attention
    q, k, v, cu = make(lens, 4, 2, torch.float16)
    ref = reference(q, k, v, lens)
    a = lens[0] - 21
    k[a:lens[0]] = value
    v[a:lens[0]] = value
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = prompt_attention(q, k, v, cu, max(lens), status=status)
    check(out, lse, ref, slice(0, a))
    check(out, lse, ref, slice(lens[0], None))
    assert not bool(torch.isfinite(out[a:lens[0]]).all()) and int(status) == 8


def test_value_seen_by_some_rows():
    """One infinite V element: the rows that see it get it in its channel only."""
    from nsn_b200.prompt import prompt_attention
    lens = [130, 700]
    q, k, v, cu = make(lens, 2, 1, torch.bfloat16)
    ref = reference(q, k, v, lens)
    for t in (77, 130 + 300):
        v[t, 0, 9] = math.inf
    out, lse = prompt_attention(q, k, v, cu, 700)
    seen = torch.zeros(830, dtype=torch.bool, device="cuda")
    seen[77:130] = True
    seen[430:] = True
    assert bool(torch.isinf(out[seen][..., 9]).all())
    clean = [t.clone() for t in ref]
    out = out.clone()
    out[seen, :, 9] = 0
    clean[0][seen, :, 9] = 0
    check(out, lse, clean)


def test_large_scores_and_equal_rows():
    """Scores in the hundreds (one token wins) and identical keys (a plain mean)."""
    from nsn_b200.prompt import prompt_attention
    lens = [300]
    q, k, v, cu = make(lens, 2, 1, torch.float16)
    check(*prompt_attention(q * 8, k, v, cu, 300), reference(q * 8, k, v, lens))
    k[:] = k[:1]
    check(*prompt_attention(q, k, v, cu, 300), reference(q, k, v, lens))


def test_rows_outside_every_sequence_and_empty_batch():
    from nsn_b200.prompt import prompt_attention
    q, k, v, cu = make([100, 30], 4, 2, torch.float16, extra=17)
    out = torch.full_like(q, 7.0)
    lse = torch.full((147, 4), 7.0, device="cuda")
    prompt_attention(q, k, v, cu, 100, out=out, lse=lse)
    check(out[:130], lse[:130], reference(q[:130], k[:130], v[:130], [100, 30]))
    assert bool((out[130:] == 7).all()) and bool((lse[130:] == 7).all())
    out, lse = prompt_attention(q[:0], k[:0], v[:0], torch.zeros(1, dtype=torch.int32, device="cuda"), 0)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)


def test_same_result_twice_and_on_another_stream():
    from nsn_b200.prompt import prompt_attention
    q, k, v, cu = make([900, 77, 1300], 8, 2, torch.bfloat16)
    a, e = prompt_attention(q, k, v, cu, 1300)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b, f = prompt_attention(q, k, v, cu, 1300)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, b) and torch.equal(e, f)


def test_captures_in_a_graph():
    from nsn_b200.prompt import prompt_attention
    lens = [333, 500]
    q, k, v, cu = make(lens, 4, 2, torch.float16)
    out, lse = prompt_attention(q, k, v, cu, 500)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        prompt_attention(q, k, v, cu, 500, out=out, lse=lse)
    out.zero_()
    graph.replay()
    check(out, lse, reference(q, k, v, lens))


def test_refusals():
    from nsn_b200 import ContractError
    from nsn_b200.prompt import prompt_attention
    q, k, v, cu = make([64], 4, 2, torch.float16)
    for bad in [dict(q=q.float()), dict(q=q[:, :3]), dict(k=k[:63]), dict(v=v.bfloat16()), dict(cu=cu.long()),
                dict(cu=cu.cpu()), dict(q=q[..., :64]), dict(q=q.cpu()), dict(k=k.transpose(1, 2)),
                dict(out=torch.empty(64, 4, 128, device="cuda")), dict(lse=torch.empty(4, 64, device="cuda"))]:
        a = dict(q=q, k=k, v=v, cu=cu, out=None, lse=None) | bad
        with pytest.raises(ContractError):
            prompt_attention(a["q"], a["k"], a["v"], a["cu"], 64, out=a["out"], lse=a["lse"])
    wide = torch.zeros((64, 4, 132), dtype=torch.float16, device="cuda")
    with pytest.raises(ContractError):
        prompt_attention(wide[..., 1:129], k, v, cu, 64)


@pytest.mark.parametrize("lens", [[40, 13], [300, 45]], ids=str)
@pytest.mark.parametrize("where", ["q", "k"])
def test_a_row_without_a_finite_score_is_nan(lens, where):
    """A row whose scores are all NaN has a NaN output and log-sum-exp, not those of a row that
    sees nothing; the other rows keep theirs."""
    from nsn_b200.prompt import prompt_attention
    q, k, v, cu = make(lens, 4, 2, torch.float16)
    ref = reference(q, k, v, lens)
    bad = torch.zeros(sum(lens), dtype=torch.bool, device="cuda")
    if where == "q":
        q[20] = math.nan
        bad[20] = True
    else:  # the second sequence's first token: every row of it sees it, its first row nothing else
        k[lens[0]] = math.nan
        bad[lens[0]:] = True
    out, lse = prompt_attention(q, k, v, cu, max(lens))
    assert bool(out[bad].isnan().all()) and bool(lse[bad].isnan().all())
    check(out, lse, ref, ~bad)


@pytest.mark.parametrize("lens", [[30], [513, 20]], ids=str)
def test_an_unknown_longest_sequence(lens):
    """max_seqlen 0 is not known: the whole call is computed."""
    from nsn_b200.prompt import prompt_attention
    q, k, v, cu = make(lens, 4, 2, torch.float16)
    out, lse = torch.full_like(q, 7.0), torch.full((sum(lens), 4), 7.0, device="cuda")
    prompt_attention(q, k, v, cu, 0, out=out, lse=lse)
    check(out, lse, reference(q, k, v, lens))


@pytest.mark.parametrize("T", [60, 200])
def test_an_output_that_rounds_past_the_type_is_reported(T):
    """V at fp16's largest value and probabilities that all round up: sum round(p) v / sum p is
    above 65520, which is infinity in fp16; the status word has to say so.

    Token 0's score is x above the others', x log2(e) = 1 - log2(1 + 5 2^-13): their p is
    1/2 + 5 2^-14, between the midpoint 1/2 + 2^-12 of two fp16 values and the upper one."""
    from nsn_b200.prompt import prompt_attention
    x = (1 - math.log2(1 + 5 * 2.0 ** -13)) / 1.4426950408889634 * math.sqrt(128)  # q . (k_0 - k_j)
    q = torch.zeros((T, 1, 128), dtype=torch.float16, device="cuda")
    k = torch.zeros_like(q)
    hi = float(torch.tensor(x, dtype=torch.float16))
    lo = float(torch.tensor((x - hi) * 1024, dtype=torch.float16))  # x = hi + lo / 1024 within 2^-20
    q[..., 0] = 1
    q[..., 1] = 1 / 1024
    k[0, 0, 0], k[0, 0, 1] = hi, lo
    v = torch.full_like(q, 65504.0)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, _ = prompt_attention(q, k, v, cu, T, status=status)
    assert bool(out[-1].isinf().all())  # the case is what it says
    assert int(status) == 8


def test_status_elsewhere_is_refused():
    from nsn_b200 import ContractError
    from nsn_b200.prompt import prompt_attention
    q, k, v, cu = make([64], 4, 2, torch.float16)
    for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, device="cuda")):
        with pytest.raises(ContractError):
            prompt_attention(q, k, v, cu, 64, status=bad)


@pytest.mark.parametrize("causal", [True, False])
def test_several_long_items_per_cta(causal):
    """More pairs of row tiles than SMs, of several K / V tiles each: S of the next item is
    issued while an item ends."""
    from nsn_b200.prompt import prompt_attention
    lens = [1500, 200, 700, 1100]
    q, k, v, cu = make(lens, 40, 8, torch.bfloat16, fused=True)
    out, lse = prompt_attention(q, k, v, cu, 1500, causal=causal)
    check(out, lse, reference(q, k, v, lens, causal))


def test_unseen_values_in_later_items():
    """Non-finite V in the shorter sequences, whose items are a CTA's second and later ones."""
    from nsn_b200.prompt import prompt_attention
    lens = [1500, 600, 450]
    q, k, v, cu = make(lens, 40, 8, torch.float16)
    ref = reference(q, k, v, lens)
    bad = torch.zeros(sum(lens), dtype=torch.bool, device="cuda")
    for first, last in ((1500 + 580, 2100), (2100 + 449, 2550)):
        v[first:last] = math.nan
        bad[first:last] = True
    out, lse = prompt_attention(q, k, v, cu, 1500)
    assert bool(out[bad].isnan().all())
    check(out, lse, ref, ~bad)
    assert bool(((lse.double() - ref[1]).abs() <= ref[3])[bad].all())  # lse does not look at V
