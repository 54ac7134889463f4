"""The shared cache and the decoder over it, against caches that share nothing."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def rows(n, h, seed, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn((h, n, 128), generator=g, device="cuda").to(dtype) for _ in range(2)]


def token(batch, hq, h, seed, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    return [torch.randn((batch, x, 128), generator=g, device="cuda").to(dtype) for x in (hq, h, h)]


def refs_hold(c):
    want = np.bincount(c.block_table.cpu().numpy().reshape(-1), minlength=c.pages)
    want[0] = 1
    assert np.array_equal(c.page_refs.cpu().numpy(), want)
    assert np.array_equal(c.n_blocks.cpu().numpy(), c.host_blocks) and np.array_equal(c.tail_len.cpu().numpy(),
                                                                                      c.host_tail)


@pytest.mark.parametrize("bits,dtype,hq", [(3, torch.float16, 8), (3, torch.bfloat16, 16), (5, torch.float16, 4)])
@pytest.mark.parametrize("prompt", [64, 64 * 5 + 17, 63])
def test_forked_sequences_decode_like_separate_ones(bits, dtype, hq, prompt):
    """Plain and shared steps over forks against an ordinary cache holding the prompt per
    sequence, across seals.  Both round K; V is fp32-restored there and rounded to dtype in the
    shared prefix, so outputs differ by V's, p's and the outputs' roundings: 4 units of dtype."""
    from nsn_b200.paged import PagedKVCache
    from nsn_b200.shared import SharedPagedKVCache
    batch, h, steps = 5, 2, 70
    k, v = rows(prompt, h, 1, dtype)
    plain = PagedKVCache(batch, h, 9, bits=bits, dtype=dtype, hq=hq)
    for b in range(batch):
        plain.prefill(b, k, v)
    shared = SharedPagedKVCache(batch, h, 9, 8 + 3 * batch, bits=bits, dtype=dtype, hq=hq)
    shared.prefill(2, k, v)
    shared.fork(2, [0, 1, 3, 4])
    refs_hold(shared)
    plan = shared.share([[2, 0, 1, 4]])  # sequence 3 outside the group
    unit = 2.0 ** (-10 if dtype == torch.float16 else -7)
    for i in range(steps):
        q, kn, vn = token(batch, hq, h, i, dtype)
        want = plain.step(q, kn, vn).float()
        got = (shared.step_shared(plan, q, kn, vn) if i % 3 else shared.step(q, kn, vn)).float()
        if not i % 3:
            plan.refresh(shared)
        assert float((got - want).abs().max()) <= 4 * unit * max(1.0, float(want.abs().max())), i
    shared.check()
    refs_hold(shared)
    for b in range(batch):
        for x, y in zip(plain.export_groups(b), shared.export_groups(b)):
            if isinstance(x, dict):
                assert torch.equal(x["codes"], y["codes"]) and all(torch.equal(s, t) for s, t in zip(x["metas"],
                                                                                                     y["metas"]))
            else:
                assert (x is None and y is None) or torch.equal(x, y)


def test_free_compact_and_reuse():
    from nsn_b200.shared import SharedPagedKVCache
    c = SharedPagedKVCache(4, 2, 12, 40, hq=4)
    for b in range(3):
        c.prefill(b, *rows(64 * (3 + 2 * b) + 9, 2, b))
    before = [c.to_bytes(b) for b in range(3)]
    c.fork(1, 3)
    c.free([0])
    refs_hold(c)
    live = c.compact()
    refs_hold(c)
    held = int((c.page_refs > 0).sum())
    assert int(live) == held and int(c.block_table.max()) < held
    assert [c.to_bytes(b) for b in (1, 2, 3)] == [before[1], before[2], before[1]]
    c.prefill(0, *rows(64 * 3 + 9, 2, 0))
    assert c.to_bytes(0) == before[0] and c.to_bytes(2) == before[2]
    refs_hold(c)
    c.load_bytes(3, before[2])
    assert c.to_bytes(3) == before[2]
    refs_hold(c)
    c.check()


def test_pool_exhaustion_is_reported():
    from nsn_b200 import ContractError
    from nsn_b200.shared import SharedPagedKVCache
    c = SharedPagedKVCache(2, 1, 8, 6, hq=2)
    c.prefill(0, *rows(64 * 3, 1, 0))
    c.check()
    c.prefill(1, *rows(64 * 3, 1, 1))
    with pytest.raises(ContractError):
        c.check()


def test_refusals():
    from nsn_b200 import ContractError
    from nsn_b200.shared import SharedPagedKVCache
    c = SharedPagedKVCache(3, 1, 4, 20, hq=2)
    c.prefill(0, *rows(70, 1, 0))
    for bad in (lambda: c.fork(0, [0]), lambda: c.fork(0, [1, 1]), lambda: c.fork([0, 1], [1, 2]), lambda: c.fork(0, 3),
                lambda: c.share([[0, 1], [1, 2]]), lambda: c.share([[]]), lambda: c.extend(0, *rows(5, 1, 0)),
                lambda: c.prefill(1, *rows(64 * 5, 1, 0)), lambda: SharedPagedKVCache(3, 1, 4, 3, hq=2),
                lambda: SharedPagedKVCache(3, 1, 4, 20, bits=4, hq=2)):
        with pytest.raises(ContractError):
            bad()


@pytest.mark.parametrize("prompt", [200, 256])
def test_shared_prompt_decoder(prompt):
    """Teacher-forced logits of samples of one prompt: the shared decoder against the batched
    decoder given the prompt per sequence, eager and replayed."""
    from transformers import LlamaConfig
    from nsn_b200 import adapter
    from nsn_b200.looped import PagedLoopedDecoder
    from nsn_b200.shared import SharedPromptDecoder
    torch.manual_seed(0)
    cfg = LlamaConfig(hidden_size=256, num_attention_heads=2, num_key_value_heads=1, head_dim=128, num_hidden_layers=2,
                      intermediate_size=512, vocab_size=320, rope_theta=10000.0)
    model = adapter.LoopedDecoder(cfg, loops=2).cuda().half().eval()
    batch = 3
    ids = torch.randint(0, 320, (prompt,), device="cuda")
    nxt = torch.randint(0, 320, (80, batch), device="cuda")
    a = PagedLoopedDecoder(model, batch, prompt + 100)
    b = SharedPromptDecoder(model, batch, prompt + 100)
    la, lb = a.prefill(ids[None].expand(batch, -1)), b.prefill(ids)
    scale = float(la.abs().max())
    # two attention roundings per layer evaluation (4 evaluations) of fp16 activations, with margin
    tol = 4 * 8 * 2.0 ** -10 * scale
    assert float((la[0] - lb).abs().max()) <= tol
    for i in range(75):
        if i == 4:
            b.capture()
        x, y = a.step(nxt[i]), (b.replay(nxt[i]) if i >= 4 else b.step(nxt[i]))
        assert float((x - y).abs().max()) <= tol, i
    b.sync_counters()
    b.release()
    b.check()
    for c in b.caches:
        refs_hold(c)


def pair(batch, prompt, groups, max_blocks=8, hq=4, dtype=torch.float16):
    """A shared cache whose sequences are forks of one prompt, a plain cache holding the prompt per
    sequence, and the plans of ``groups``."""
    from nsn_b200.paged import PagedKVCache
    from nsn_b200.shared import SharedPagedKVCache
    h = 2
    k, v = rows(prompt, h, 1, dtype)
    plain = PagedKVCache(batch, h, max_blocks, dtype=dtype, hq=hq)
    for b in range(batch):
        plain.prefill(b, k, v)
    shared = SharedPagedKVCache(batch, h, max_blocks, max_blocks * batch + 1, dtype=dtype, hq=hq)
    shared.prefill(0, k, v)
    shared.fork(0, range(1, batch))
    return plain, shared, [shared.share(g) for g in groups]


def agree(got, want, unit=2.0 ** -10):
    """As test_forked_sequences_decode_like_separate_ones: 4 units of dtype."""
    assert float((got.float() - want.float()).abs().max()) <= 4 * unit * max(1.0, float(want.float().abs().max()))


@pytest.mark.parametrize("host", [False, True])
def test_a_plan_follows_plain_steps(host):
    """Plain steps seal blocks into pages that the plan was made before."""
    plain, shared, (plan,) = pair(3, 200, [[[0, 1, 2]]])
    for i in range(150):
        q, kn, vn = token(3, 4, 2, i)
        want = plain.step(q, kn, vn)
        if host:
            packed = torch.cat([x.reshape(-1) for x in (q, kn, vn)]).cpu().pin_memory()
            out, done = torch.empty(3 * 4 * 128, dtype=q.dtype).pin_memory(), torch.cuda.Event()
            shared.step_host(packed, out, done)
            done.synchronize()
        else:
            shared.step(q, kn, vn)
    q, kn, vn = token(3, 4, 2, 999)
    agree(shared.step_shared(plan, q, kn, vn), plain.step(q, kn, vn))
    refs_hold(shared)


def test_two_plans_take_turns():
    """Two plans of one cache on alternate steps: every second plan's steps never seal."""
    plain, shared, plans = pair(4, 130, [[[0, 1, 2, 3]], [[0, 1], [2, 3]]])
    for i in range(260):
        q, kn, vn = token(4, 4, 2, i)
        agree(shared.step_shared(plans[i % 2], q, kn, vn), plain.step(q, kn, vn))
    refs_hold(shared)


def test_a_plan_follows_extend():
    """A sequence outside the batch's rhythm: more blocks appended behind its prefix."""
    plain, shared, (plan,) = pair(2, 128, [[[0, 1]]])
    k, v = rows(64 * 3, 2, 9)
    shared.extend(1, k, v)
    k0, v0 = rows(128, 2, 1)
    plain.prefill(1, torch.cat([k0, k], 1), torch.cat([v0, v], 1))
    q, kn, vn = token(2, 4, 2, 5)
    agree(shared.step_shared(plan, q, kn, vn), plain.step(q, kn, vn))


def test_a_captured_shared_step_among_eager_ones():
    """Replays and eager steps of both kinds in turn: each finds the pages that the other took."""
    plain, shared, (plan,) = pair(3, 70, [[[0, 1, 2]]])
    q, kn, vn = token(3, 4, 2, 0)
    out = torch.empty_like(q)
    snap = shared.host_blocks.copy(), shared.host_tail.copy()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        shared.step_shared(plan, q, kn, vn, out=out)
    shared.host_blocks[:], shared.host_tail[:] = snap
    for i in range(300):
        for x, y in zip((q, kn, vn), token(3, 4, 2, i)):
            x.copy_(y)
        want = plain.step(q, kn, vn)
        if 60 <= i < 200 or i >= 280:  # 140 plain steps, then replays again, then shared steps
            agree(shared.step(q, kn, vn) if i < 200 else shared.step_shared(plan, q, kn, vn), want)
        else:
            graph.replay()
            agree(out, want)
            shared.host_blocks[:] = shared.n_blocks.cpu().numpy()
            shared.host_tail[:] = shared.tail_len.cpu().numpy()
    refs_hold(shared)
    del graph



def test_a_plan_ends_with_what_its_sequences_held():
    from nsn_b200 import ContractError
    from nsn_b200.shared import SharedPagedKVCache
    args = token(3, 4, 2, 0)
    for change in (lambda c: c.free([2]), lambda c: c.fork(0, [1]), lambda c: c.prefill(1, *rows(200, 2, 4)),
                   lambda c: c.compact(), lambda c: c.load_bytes(1, c.to_bytes(0))):
        _, shared, (plan,) = pair(3, 200, [[[0, 1, 2]]])
        shared.step_shared(plan, *args)
        change(shared)
        before = shared.lengths()
        with pytest.raises(ContractError):
            shared.step_shared(plan, *args)
        assert torch.equal(shared.lengths(), before)
        shared.step_shared(shared.share([[0, 1, 2]]), *args)
    _, other, _ = pair(3, 200, [])
    with pytest.raises(ContractError):  # a plan of another cache
        other.step_shared(shared.share([[0, 1, 2]]), *args)


def test_attend_and_seal_take_pages_too():
    """The pair that step runs in one call, over several seals, against an ordinary cache."""
    plain, shared, _ = pair(3, 70, [])
    for i in range(200):
        args = token(3, 4, 2, i)
        want, got = plain.attend(*args).clone(), shared.attend(*args)
        plain.seal(1)
        shared.seal(1)
        assert torch.equal(got, want), i
    refs_hold(shared)
    assert [shared.to_bytes(b) for b in range(3)] == [plain.to_bytes(b) for b in range(3)]
    shared.check()


def test_import_checks_what_it_loads():
    """Groups of another head count, wrong headers, missing blocks: refused as by PagedKVCache."""
    from nsn_b200 import ContractError
    from nsn_b200.shared import SharedPagedKVCache
    c = SharedPagedKVCache(2, 2, 6, 20, hq=4)
    one = SharedPagedKVCache(2, 1, 6, 20, hq=2)
    c.prefill(0, *rows(64 * 2 + 5, 2, 0))
    one.prefill(0, *rows(64 * 2 + 5, 1, 0))
    kg, kt, vg, vt = c.export_groups(0)
    kg1, _, vg1, _ = one.export_groups(0)
    wrong = dict(kg, headers=kg["headers"].clone())
    wrong["headers"][0, 1, 0, 8] ^= 1
    short = {**vg, "codes": vg["codes"][:, :, :1]}
    for bad in ((kg1, kt, vg1, vt), (wrong, kt, vg, vt), (kg, kt, dict(vg, headers=wrong["headers"]), vt),
                (kg, kt, short, vt)):
        with pytest.raises(ContractError):
            c.import_groups(1, *bad)
    c.import_groups(1, kg, kt, vg, vt)
    assert c.to_bytes(1) == c.to_bytes(0)


def test_a_refused_load_leaves_the_sequence():
    from nsn_b200 import ContractError
    from nsn_b200.shared import SharedPagedKVCache
    c = SharedPagedKVCache(2, 2, 4, 20, hq=4)
    big = SharedPagedKVCache(1, 2, 6, 20, hq=4)
    c.prefill(1, *rows(64 * 2 + 5, 2, 0))
    big.prefill(0, *rows(64 * 4 + 1, 2, 1))
    kg, kt, vg, vt = big.export_groups(0)
    before = c.to_bytes(1)
    k, v = rows(100, 2, 3)
    for bad in (lambda: c.prefill(1, *rows(64 * 5, 2, 0)), lambda: c.prefill(1, k, v[:, :99]),
                lambda: c.prefill(1, k[:1], v[:1]), lambda: c.prefill(1, k[..., :64], v[..., :64]),
                lambda: c.prefill(1, k.cpu(), v.cpu()),
                lambda: c.import_groups(1, kg, torch.cat([kt] * 64, 2), vg, torch.cat([vt] * 64, 2)),
                lambda: c.import_groups(1, kg, kt, None, vt), lambda: c.import_groups(1, kg, kt[:, :1], vg, vt[:, :1])):
        with pytest.raises(ContractError):
            bad()
        assert c.to_bytes(1) == before
    refs_hold(c)


def test_a_full_sequence_refuses_the_shared_step():
    """The step that would fill the last tail is refused before anything changes, as step's is."""
    from nsn_b200._lib import NativeError
    _, shared, (plan,) = pair(2, 64 * 3 + 60, [[[0, 1]]], max_blocks=3)
    args = token(2, 4, 2, 0)
    for _ in range(3):
        shared.step_shared(plan, *args)
    for call in (lambda: shared.step_shared(plan, *args), lambda: shared.step(*args)):
        with pytest.raises(NativeError):
            call()
        assert shared.host_blocks.tolist() == [3, 3] and shared.host_tail.tolist() == [63, 63]
        refs_hold(shared)
    shared.check()


@pytest.mark.parametrize("prompt,new", [(200, 50), (128, 1), (64 * 3 + 63, 130)])
def test_a_new_turn_after_a_cached_prompt(prompt, new):
    """The new tokens' queries over sealed blocks, cached tail and new tokens: prompt attention over
    tail and new tokens (the tail's rows are dropped), merged with the sealed blocks.

    Bound: the output's rounding u |o|, the probabilities' u sum p |v| in both parts, the own
    part's rounding, at most u sum p |v| again, and scores as in tests/test_gpu_prompt.py."""
    import test_gpu_prefix as R
    from nsn_b200.prefix import prefix_attention
    from nsn_b200.prompt import prompt_attention
    from nsn_b200.shared import SharedPagedKVCache
    h, hq, u = 2, 8, 2.0 ** -11
    c = SharedPagedKVCache(1, h, 6, 12, hq=hq)
    c.prefill(0, *rows(prompt, h, 3))
    k, v = rows(new, h, 4)
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn((new, hq, 128), generator=g, device="cuda").half()
    n, t = int(c.host_blocks[0]), int(c.host_tail[0])
    own_k, own_v = (torch.cat([tail[0, :, :t], x], 1).transpose(0, 1) for tail, x in ((c.k_tail, k), (c.v_tail, v)))
    own_q = torch.cat([q.new_zeros((t, hq, 128)), q])
    cu = torch.tensor([0, t + new], dtype=torch.int32, device="cuda")
    o, e = prompt_attention(own_q, own_k, own_v, cu, t + new)
    out, _ = prefix_attention(q, c.records, c.block_table[:1, :n], o_part=o[t:].float(), lse_part=e[t:].contiguous())
    pages = c.block_table[0, :n].long()
    sealed = [R.rows_of({a: b[:, pages] if torch.is_tensor(b) else b for a, b in p.items()}, 3, torch.float16)
              for p in (c.k_pool, c.v_pool)]
    kk, vv = (torch.cat([s.reshape(h, 64 * n, 128), x.transpose(0, 1)], 1).double() for s, x in zip(sealed,
                                                                                                    (own_k, own_v)))
    seen = torch.arange(prompt + new, device="cuda")[None] <= prompt + torch.arange(new, device="cuda")[:, None]
    for j in range(hq):
        x = q[:, j].double() @ kk[j // 4].T / 128 ** 0.5
        dx = 2.0 ** -20 * (1 + (q[:, j].double().abs() @ kk[j // 4].abs().T).amax(1, keepdim=True) / 128 ** 0.5)
        p = torch.softmax(x.masked_fill(~seen, -float("inf")), 1)
        want, big = p @ vv[j // 4], p @ vv[j // 4].abs()
        tol = u * (want.abs() + 2 * big) * 1.01 + 5 * dx * big + (prompt + new) * 2.0 ** -25 * vv.abs().amax()
        assert bool(((out[:, j].double() - want).abs() <= tol).all()), j
