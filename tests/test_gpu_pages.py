"""Page operations against a plain host model of the table, the counts and the pool."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def state(batch, mb, pages, h=2, seed=0, reserved=1):
    """A random valid cache: sealed pages (some shared), reserved pages, tails."""
    rng = np.random.default_rng(seed)
    n = rng.integers(0, mb + 1, batch).astype(np.int32)
    free = list(rng.permutation(np.arange(1, pages)))
    table = np.zeros((batch, mb), np.int32)
    for b in range(batch):
        for i in range(min(mb, n[b] + reserved)):
            share = b and i < n[b] and i < n[b - 1] and rng.random() < 0.4
            if share:
                table[b, i] = table[b - 1, i]
            elif free:
                table[b, i] = free.pop()
            else:
                n[b] = min(n[b], i)
    refs = np.bincount(table.reshape(-1), minlength=pages).astype(np.int32)
    refs[0] = 1
    tl = rng.integers(0, 64, batch).astype(np.int32)
    tails = [rng.standard_normal((batch, h, 64, 128)).astype(np.float16) for _ in range(2)]
    return dict(table=table, n=n, tl=tl, refs=refs, kt=tails[0], vt=tails[1])


def host_fork(s, src, dst):
    for a, b in zip(src, dst):
        for p in s["table"][b]:
            if p > 0:
                s["refs"][p] -= 1
        row = np.where(np.arange(s["table"].shape[1]) < s["n"][a], s["table"][a], 0)
        for p in row:
            if p > 0:
                s["refs"][p] += 1
        s["table"][b], s["n"][b], s["tl"][b] = row, s["n"][a], s["tl"][a]
        t = s["tl"][a]
        s["kt"][b, :, :t], s["vt"][b, :, :t] = s["kt"][a, :, :t], s["vt"][a, :, :t]


def same(s, d):
    for name, t in d.items():
        assert np.array_equal(t.cpu().numpy(), s[name]), name


@pytest.mark.parametrize("dtype", ["float16", "int16"])
@pytest.mark.parametrize("batch,mb,src,dst", [
    (2, 1, [0], [1]), (4, 5, [0, 0, 0], [1, 2, 3]), (9, 130, [3, 7, 3, 0], [1, 8, 2, 5]), (64, 300, [5] * 40,
                                                                                         list(range(20, 60)))])
def test_fork(batch, mb, src, dst, dtype):
    from nsn_b200.pages import fork_sequences
    s = state(batch, mb, batch * mb + 1, seed=batch)
    d = {k: dev(v) for k, v in s.items()}
    bf = dtype == "int16"  # the same bits as bf16 tails
    kt, vt = (d[x].view(torch.bfloat16) if bf else d[x] for x in ("kt", "vt"))
    fork_sequences(d["table"], d["n"], d["tl"], d["refs"], kt, vt, dev(np.int32(src)), dev(np.int32(dst)))
    host_fork(s, src, dst)
    same(s, d)


def test_fork_skips_bad_numbers():
    from nsn_b200.pages import fork_sequences, free_sequences
    s = state(3, 4, 13)
    d = {k: dev(v) for k, v in s.items()}
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    fork_sequences(d["table"], d["n"], d["tl"], d["refs"], d["kt"], d["vt"], dev(np.int32([0, 7, -1])),
                   dev(np.int32([3, 1, 2])), status=st)
    same(s, d)
    assert int(st) == 128
    st.zero_()
    free_sequences(d["table"], d["n"], d["tl"], d["refs"], dev(np.int32([3, -1])), status=st)
    same(s, d)
    assert int(st) == 128


def test_free():
    from nsn_b200.pages import free_sequences
    s = state(7, 20, 141, seed=3)
    d = {k: dev(v) for k, v in s.items()}
    free_sequences(d["table"], d["n"], d["tl"], d["refs"], dev(np.int32([2, 6, 2])))
    for b in (2, 6):
        for p in s["table"][b]:
            if p > 0:
                s["refs"][p] -= 1
        s["table"][b] = s["n"][b] = s["tl"][b] = 0
    same(s, d)


@pytest.mark.parametrize("batch,mb,pages,ahead", [(1, 1, 2, 1), (5, 8, 60, 1), (64, 40, 2600, 1), (30, 90, 2701, 3),
                                                  (1500, 3, 4600, 2), (4, 50, 30, 7)])
def test_reserve(batch, mb, pages, ahead):
    from nsn_b200.pages import reserve_pages
    s = state(batch, mb, pages, seed=batch + ahead, reserved=0)
    d = {k: dev(s[k]) for k in ("table", "n", "refs")}
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    reserve_pages(d["table"], d["n"], d["refs"], ahead, status=st)
    free = iter([p for p in range(1, pages) if s["refs"][p] == 0])
    short = False
    for b in range(batch):
        for i in range(s["n"][b], min(mb, s["n"][b] + ahead)):
            if s["table"][b, i] == 0:
                p = next(free, None)
                short |= p is None
                if p is not None:
                    s["table"][b, i], s["refs"][p] = p, 1
    same(s, d)
    assert int(st) == (64 if short else 0)
    reserve_pages(d["table"], d["n"], d["refs"], ahead)  # nothing left to do, or nothing to give
    same(s, d)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,mb,pages,seed", [(1, 1, 1, 0), (1, 1, 2, 1), (3, 10, 64, 2), (8, 100, 801, 3),
                                                 (20, 150, 6007, 4), (2, 6, 3000, 5)])
def test_compact(batch, mb, pages, seed, in_place):
    from nsn_b200.pages import compact_pages
    s = state(batch, mb, pages, seed=seed)
    rng = np.random.default_rng(seed)
    rec = rng.integers(0, 256, (3, pages, 7680), dtype=np.uint8) if pages < 1000 else \
        np.broadcast_to(np.arange(3 * pages, dtype=np.int32).reshape(3, pages, 1), (3, pages, 32)).copy().view(np.uint8)
    norm = rng.standard_normal((3, pages, 64)).astype(np.float16)
    used = s["refs"] > 0
    used[0] = True
    live = int(used.sum())
    src = [p for p in range(pages) if used[p] and p >= live]
    dst = [p for p in range(pages) if not used[p] and p < live]
    to = np.arange(pages)
    to[src] = dst
    table, refs = dev(s["table"]), dev(s["refs"])
    d = [dev(rec), dev(norm)]
    t, r, n = compact_pages(d, table, refs, table_out=table if in_place else None,
                            refs_out=refs if in_place else None)
    for x, got in ((rec, d[0]), (norm, d[1])):
        x[:, dst] = x[:, src]
        assert np.array_equal(got.cpu().numpy(), x)
    want = np.zeros_like(s["refs"])
    want[to[used]] = s["refs"][used]
    assert int(n) == live and np.array_equal(t.cpu().numpy(), to[s["table"]])
    assert np.array_equal(r.cpu().numpy(), want)
    if not in_place:
        assert np.array_equal(table.cpu().numpy(), s["table"]) and np.array_equal(refs.cpu().numpy(), s["refs"])


def test_copy_pages():
    from nsn_b200.pages import copy_pages
    rng = np.random.default_rng(0)
    a = rng.integers(0, 256, (2, 50, 7680), dtype=np.uint8)
    b = rng.standard_normal((2, 60, 64)).astype(np.float16)
    da, db = dev(a), dev(b)[:, 10:]
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    copy_pages([da, db], dev(np.int32([1, 9, 1, 50])), dev(np.int32([49, 0, 30, 2])), status=st)
    for s_, t_ in ((1, 49), (9, 0), (1, 30)):
        a[:, t_] = a[:, s_]
        b[:, 10 + t_] = b[:, 10 + s_]
    assert np.array_equal(da.cpu().numpy(), a) and np.array_equal(db.cpu().numpy(), b[:, 10:]) and int(st) == 128


def test_refusals():
    from nsn_b200 import ContractError
    from nsn_b200 import pages as P
    s = state(3, 4, 13)
    d = {k: dev(v) for k, v in s.items()}
    one, two = dev(np.int32([0])), dev(np.int32([1, 2]))
    for bad in [dict(table=d["table"].long()), dict(n=d["n"][:2]), dict(kt=d["kt"].float()), dict(src=two),
                dict(vt=d["vt"][:2]), dict(refs=d["refs"].cpu())]:
        a = dict(d, src=one, dst=dev(np.int32([1]))) | bad
        with pytest.raises(ContractError):
            P.fork_sequences(a["table"], a["n"], a["tl"], a["refs"], a["kt"], a["vt"], a["src"], a["dst"])
    rec = torch.zeros((2, 13, 7680), dtype=torch.uint8, device="cuda")
    with pytest.raises(ContractError):
        P.compact_pages([], d["table"], d["refs"])
    with pytest.raises(ContractError):
        P.compact_pages([rec], d["table"], d["refs"][:12])
    with pytest.raises(ContractError):
        P.compact_pages([rec, rec[:, :12]], d["table"], d["refs"])
    with pytest.raises(ContractError):
        P.copy_pages([rec], one, two)


def test_fork_drops_entries_outside_the_pool():
    """A source entry that names no page of the pool is not handed on: 0 in the target, and a status."""
    from nsn_b200.pages import fork_sequences
    s = state(3, 6, 19, seed=1)
    s["n"][0] = 5
    s["table"][0, 1], s["table"][0, 3] = 19, -4
    d = {k: dev(v) for k, v in s.items()}
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    fork_sequences(d["table"], d["n"], d["tl"], d["refs"], d["kt"], d["vt"], dev(np.int32([0])), dev(np.int32([2])),
                   status=st)
    for p in s["table"][2]:
        s["refs"][p] -= p > 0
    row = np.where(np.arange(6) < 5, s["table"][0], 0)
    row[[1, 3]] = 0
    for p in row:
        s["refs"][p] += p > 0
    s["table"][2], s["n"][2], s["tl"][2] = row, 5, s["tl"][0]
    s["kt"][2, :, :s["tl"][0]], s["vt"][2, :, :s["tl"][0]] = s["kt"][0, :, :s["tl"][0]], s["vt"][0, :, :s["tl"][0]]
    same(s, d)
    assert int(st) == 128


def test_free_reports_entries_outside_the_pool():
    from nsn_b200.pages import free_sequences
    for value in (13, -1):
        s = state(3, 4, 13, seed=2)
        s["table"][1, 3] = value
        d = {k: dev(v) for k, v in s.items()}
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        free_sequences(d["table"], d["n"], d["tl"], d["refs"], dev(np.int32([1])), status=st)
        for p in s["table"][1, :3]:
            s["refs"][p] -= p > 0
        s["table"][1] = s["n"][1] = s["tl"][1] = 0
        same(s, d)
        assert int(st) == 128


def test_status_elsewhere_is_refused():
    from nsn_b200 import ContractError
    from nsn_b200 import pages as P
    s = state(3, 4, 13)
    d = {k: dev(v) for k, v in s.items()}
    rec, one, two = torch.zeros((2, 13, 64), dtype=torch.uint8, device="cuda"), dev(np.int32([0])), dev(np.int32([1]))
    bad = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: P.fork_sequences(d["table"], d["n"], d["tl"], d["refs"], d["kt"], d["vt"], one, two, status=bad),
                 lambda: P.free_sequences(d["table"], d["n"], d["tl"], d["refs"], one, status=bad),
                 lambda: P.reserve_pages(d["table"], d["n"], d["refs"], status=bad),
                 lambda: P.copy_pages([rec], one, two, status=bad),
                 lambda: P.compact_pages([rec], d["table"], d["refs"], status=bad)):
        with pytest.raises(ContractError):
            call()
    same(s, d)


def test_workspace_elsewhere_is_refused():
    from nsn_b200 import ContractError
    from nsn_b200.pages import compact_pages
    s = state(3, 4, 13)
    table, refs, rec = dev(s["table"]), dev(s["refs"]), torch.zeros((2, 13, 64), dtype=torch.uint8, device="cuda")
    big = torch.empty(1 << 16, dtype=torch.uint8)
    for bad in (big, big.cuda()[::2]):
        with pytest.raises(ContractError):
            compact_pages([rec], table, refs, ws=bad)
