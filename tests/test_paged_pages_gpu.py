"""GPU tests of page_fork, page_free and page_compact against plain Python
restatements of include/bml_attn.h: whole numbers and rows that only move, so
everything is compared bit for bit."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


class State:
    """Random requests on shuffled pages, some of which share full pages."""

    def __init__(self, lens, page, idle=0, spare=6, share=True, seed=0, wide=2):
        rng = np.random.default_rng(seed)
        held = [-(-t // page) for t in lens]
        self.page, self.n = page, len(lens) + idle
        self.n_pages = sum(held) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((self.n, max(held + [1]) + wide), -1)
        self.shared = np.zeros(self.n_pages, int)
        at = 0
        for i, k in enumerate(held):
            both = 0
            if share and i and rng.random() < 0.6:
                j = int(rng.integers(0, i))
                both = int(rng.integers(0, min(lens[i], lens[j]) // page + 1))
                self.table[i, :both] = self.table[j, :both]
                self.shared[self.table[i, :both]] += 1
            self.table[i, both:k] = order[at:at + k - both]
            at += k - both
        self.lens, self.owned = list(lens) + [0] * idle, held + [0] * idle
        self.free, self.used = order, at

    def check(self):
        """The list's taken part holds every held page once, shared counts the rest."""
        held = [p for i in range(self.n) for p in self.table[i, :self.owned[i]]]
        assert sorted(set(held)) == sorted(self.free[:self.used])
        assert sorted(self.free) == list(range(self.n_pages))
        count = np.bincount(held, minlength=self.n_pages) if held else np.zeros(self.n_pages, int)
        assert (self.shared == np.maximum(count - 1, 0)).all()


def want_free(s, keep):
    lens, owned, shared, status = list(s.lens), list(s.owned), s.shared.copy(), [0] * s.n
    count = np.zeros(s.n_pages, int)
    for i, k in enumerate(keep):
        if k < 0:
            continue
        t = min(lens[i], k)
        if t < lens[i] and t % s.page and s.shared[s.table[i, t // s.page]] > 0:
            status[i] = 8
            continue
        stay = min(owned[i], -(-t // s.page))
        for p in s.table[i, stay:owned[i]]:
            count[p] += 1
        lens[i], owned[i] = t, stay
    gone = count > s.shared
    shared = np.where(gone, 0, s.shared - count)
    taken = s.free[:s.used]
    free = np.concatenate([taken[~gone[taken]], taken[gone[taken]], s.free[s.used:]])
    return lens, owned, shared, free, s.used - int(gone[taken].sum()), status


def call_free(s, keep, **kw):
    import bml_b200
    return bml_b200.page_free(ints(keep), ints(s.lens), ints(s.owned), ints(s.table), s.page, ints(s.shared),
                              ints(s.free), ints([s.used]), **kw)


@pytest.mark.parametrize("seed", range(12))
def test_free(cuda, seed):
    rng = np.random.default_rng(100 + seed)
    n, page = [1, 2, 7, 40, 300, 1500][seed % 6], [16, 64, 1024][seed % 3]
    lens = [int(x) for x in rng.integers(0, page * (9 if n > 100 else 40), n)]
    s = State(lens, page, idle=seed % 3, seed=seed)
    for step in range(4):
        s.check()
        keep = [int(rng.choice([-1, 0, a, a // 2, a // 2 // page * page, a + 100])) for a in s.lens]
        p = call_free(s, keep)
        want = want_free(s, keep)
        assert [x.tolist() for x in (p.lens, p.owned, p.shared, p.free_pages)] == [list(x) for x in want[:4]]
        assert p.free_used.tolist() == [want[4]] and p.status.tolist() == want[5] and p.block_table is None
        s.lens, s.owned, s.shared, s.free, s.used = want[0], want[1], want[2], want[3], want[4]


def test_free_refuses_inside_a_shared_page(cuda):
    import bml_b200
    s = State([40], 16, idle=1, share=False)
    s.table[1, :2], s.lens[1], s.owned[1] = s.table[0, :2], 32, 2
    s.shared[s.table[0, :2]] = 1
    p = call_free(s, [-1, 20])
    assert p.status.tolist() == [0, 8] and p.lens.tolist() == [40, 32] and p.owned.tolist() == [3, 2]
    with pytest.raises(bml_b200.PageRefused):
        p.check()
    p = call_free(s, [35, 16])  # the part-filled page is its own; a page's end is fine
    p.check()
    assert p.lens.tolist() == [35, 16] and p.owned.tolist() == [3, 1] and p.free_used.tolist() == [3]
    # both holders at once: refused by what is shared before the call
    assert call_free(s, [0, 20]).status.tolist() == [0, 8]


def test_free_of_state_that_does_not_hold_together(cuda):
    """Tables, counts and lists out of bounds: nothing outside the arrays is touched."""
    import bml_b200
    big = 0x7fffffff
    p = bml_b200.page_free(ints([0, 0, 0, 5, -1]), ints([100, -5, 20, 30, 40]), ints([9, 2, -3, big, 2]),
                           ints([[5, -1, big, 5, 5, 7, 0, 0, 9]] * 5), 16, ints([0, 3, -4, 0, 0, 0, 0, 0]),
                           ints([1, -7, big, 5, 5, 0, 2]), ints([big]))
    assert p.lens.tolist() == [0, -5, 20, 30, 40] and p.owned.tolist() == [0, 2, -3, big, 2]
    assert p.free_used.tolist() == [4] and p.shared.tolist() == [0, 3, 0, 0, 0, 0, 0, 0]
    assert p.free_pages.tolist() == [1, -7, big, 2, 5, 5, 0]
    p = bml_b200.page_free(ints([0]), ints([5]), ints([1]), ints([[0]]), 16, ints([0]), ints([]), ints([0]))
    assert p.free_pages.numel() == 0 and p.free_used.tolist() == [0] and p.owned.tolist() == [0]


def want_fork(s, src, dst, pools):
    lens, owned, shared, table = list(s.lens), list(s.owned), s.shared.copy(), s.table.copy()
    out, named, cum, granted, status = [p.clone() for p in pools], set(), 0, 0, []
    for a, d in zip(src, dst):
        ok = 0 <= a < s.n and 0 <= d < s.n and d not in named and s.owned[d] == 0 and s.lens[d] == 0
        if 0 <= d < s.n:
            named.add(d)
        t = s.lens[a] if ok else 0
        if not ok or s.owned[a] < -(-t // s.page):
            status.append(2)
            continue
        full, rest = t // s.page, t % s.page
        if rest:
            cum += 1
            if s.used + cum > len(s.free):
                status.append(1)
                continue
            granted = cum
            fresh = int(s.free[s.used + cum - 1])
            for p, o in zip(pools, out):
                o[:, fresh, :rest] = p[:, s.table[a, full], :rest]
            table[d, full] = fresh
        table[d, :full] = s.table[a, :full]
        shared[s.table[a, :full]] += 1
        lens[d], owned[d] = t, full + (rest > 0)
        status.append(0)
    return lens, owned, shared, s.used + granted, status, table, out


def pools_of(s, layers, kv, d, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(layers, s.n_pages, s.page, kv, d, device="cuda", generator=g).to(DT[dt]) for _ in "kv"]


def check_fork(s, src, dst, pools, **kw):
    import bml_b200
    want = want_fork(s, src, dst, pools)
    table = ints(s.table)
    p = bml_b200.page_fork(*pools, ints(src), ints(dst), ints(s.lens), ints(s.owned), table, ints(s.shared), ints(s.free),
                           ints([s.used]), **kw)
    torch.cuda.synchronize()
    assert [x.tolist() for x in (p.lens, p.owned, p.shared, p.free_used, p.status)] == [
        want[0], want[1], list(want[2]), [want[3]], want[4]]
    assert (table.cpu().numpy() == want[5]).all()
    for a, b in zip(pools, want[6]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    return p, want


@pytest.mark.parametrize("dt,kv,d", [("bf16", 8, 128), ("f16", 4, 64), ("f32", 3, 64), ("f16", 1, 6), ("f32", 2, 3)])
@pytest.mark.parametrize("seed", range(4))
def test_fork(cuda, dt, kv, d, seed):
    rng = np.random.default_rng(seed)
    page = [16, 64, 128, 32][seed]
    n, m = [1, 5, 30, 3][seed], [8, 1, 40, 0][seed]
    lens = [int(x) for x in rng.integers(0, 5 * page, n)]
    lens[0] = [3, page, 2 * page + 1, 0][seed]
    s = State(lens, page, idle=m + 2, spare=m + 1, seed=seed)
    src = rng.integers(0, n, m)
    dst = n + rng.permutation(m + 2)[:m]
    check_fork(s, [int(x) for x in src], [int(x) for x in dst], pools_of(s, [1, 3, 2, 5][seed], kv, d, dt))


def test_fork_refusals(cuda):
    """A page short, rows named twice, busy, outside; an empty row and one onto itself."""
    import bml_b200
    s = State([20, 16, 5, 37], 16, idle=8, spare=2, share=False)
    src = [0, 1, 2, 3, 3, -1, 99, 0, 5, 11, 0]
    dst = [4, 5, 6, 7, 4, 8, 8, 99, 9, 11, 2]
    p, want = check_fork(s, src, dst, pools_of(s, 2, 2, 64, "bf16"))
    assert want[4] == [0, 0, 0, 1, 2, 2, 2, 2, 0, 0, 2]
    with pytest.raises(bml_b200.OutOfPages):
        p.check()
    s.owned[1] = 0      # its pages do not hold its positions
    assert check_fork(s, [1], [5], pools_of(s, 1, 2, 64, "bf16"))[1][4] == [2]


def test_fork_of_state_that_does_not_hold_together(cuda):
    import bml_b200
    big = 0x7fffffff
    k, v = (torch.randn(2, 4, 16, 2, 64, device="cuda") for _ in "kv")
    k0 = k.clone()
    table = ints([[-1, big, 3], [0, 1, 2], [-1, -1, -1], [-1, -1, -1], [-1, -1, -1], [-1, -1, -1]])
    p = bml_b200.page_fork(k, v, ints([0, 1, 1, 1]), ints([2, 3, 4, 5]), ints([40, -3, 0, 0, 0, 0]), ints([3, 1, 0, 0, 0, 0]),
                           table, ints([0] * 4), ints([0, -5, big]), ints([-9]))
    assert p.status.tolist() == [0, 2, 2, 2] and p.free_used.tolist() == [1] and p.shared.tolist() == [0, 0, 0, 0]
    assert table[2].tolist() == [-1, big, 0]
    assert torch.equal(k[:, 1:], k0[:, 1:]) and torch.equal(k[:, 0, :8], k0[:, 3, :8]) and torch.equal(k[:, 0, 8:], k0[:, 0, 8:])
    p = bml_b200.page_fork(k, v, ints([0]), ints([2]), ints([40, 0, 0]), ints([3, 0, 0]), ints([[1, 2, 3]] * 3), ints([0] * 4),
                           ints([0, -5, big]), ints([1]))   # the free list's page is outside the pool: nothing is copied
    assert p.status.tolist() == [0] and p.free_used.tolist() == [2]


@pytest.mark.parametrize("dt,kv,d", [("bf16", 8, 128), ("f16", 4, 64), ("f32", 1, 3), ("f16", 1, 7)])
@pytest.mark.parametrize("seed", range(5))
def test_compact(cuda, dt, kv, d, seed):
    import bml_b200
    rng = np.random.default_rng(seed)
    page, n = [16, 64, 32, 16, 128][seed], [1, 6, 25, 3, 2][seed]
    lens = [int(x) for x in rng.integers(0, 6 * page, n)]
    if seed == 3:
        lens = [0, 0, 0]
    s = State(lens, page, idle=seed % 2, spare=[0, 9, 60, 4, 1][seed], seed=seed)
    pools = pools_of(s, [1, 3, 2, 2, 4][seed], kv, d, dt)
    before = [p.clone() for p in pools]
    live = sorted(set(int(p) for i in range(s.n) for p in s.table[i, :s.owned[i]]))
    h = len(live)
    move = dict(zip([p for p in live if p >= h], [p for p in range(h) if p not in set(live)]))
    u = bml_b200.page_compact(*pools, ints(s.owned), ints(s.table), ints(s.shared))
    torch.cuda.synchronize()
    table, shared = s.table.copy(), np.zeros(s.n_pages, int)
    for i in range(s.n):
        table[i, :s.owned[i]] = [move.get(p, p) for p in table[i, :s.owned[i]]]
    for p in live:
        shared[move.get(p, p)] = s.shared[p]
    assert (u.block_table.cpu().numpy() == table).all() and u.shared.tolist() == list(shared)
    assert u.free_pages.tolist() == list(range(s.n_pages)) and u.free_used.tolist() == [h]
    assert u.lens is None and u.owned is None and u.status is None
    u.check()
    for p, b in zip(pools, before):
        for a, c in move.items():
            b[:, c] = b[:, a]
        assert torch.equal(p.view(torch.uint8), b.view(torch.uint8))


def test_compact_of_a_large_pool(cuda):
    """More pages than the bookkeeping CTAs have threads, and entries outside the pool."""
    import bml_b200
    rng = np.random.default_rng(0)
    n_pages, held = 30011, 9000
    order = rng.permutation(n_pages)[:held]
    table = np.full((30, 400), 0x7fffffff)
    table[:, :300] = order.reshape(30, 300)
    pools = [torch.arange(n_pages, device="cuda", dtype=torch.float32)[None, :, None, None, None].repeat(1, 1, 16, 1, 2) for _ in "kv"]
    u = bml_b200.page_compact(*pools, ints([301] * 30), ints(table), ints(np.arange(n_pages)))
    new = u.block_table.cpu().numpy()
    assert (new[:, 300:] == 0x7fffffff).all() and u.free_used.tolist() == [held]
    assert sorted(new[:, :300].flatten()) == list(range(held))
    for p in pools:
        assert torch.equal(p[0, new[:, :300].flatten(), 0, 0, 0].cpu(), torch.from_numpy(order).float())
    assert (u.shared.cpu().numpy()[new[:, :300].flatten()] == order).all() and int(u.shared[held:].sum()) == 0


def test_streams_graphs_and_both_ways(cuda, monkeypatch):
    """The same bits on another stream, in a replayed graph and through ctypes."""
    import bml_b200
    import bml_b200.paged as P
    s = State([100, 37, 64, 5], 16, idle=3, spare=9, seed=4)
    pools = pools_of(s, 2, 2, 64, "bf16")
    a = dict(lens=ints(s.lens), owned=ints(s.owned), table=ints(s.table), shared=ints(s.shared), free=ints(s.free), used=ints([s.used]),
             keep=ints([0, 16, -1, 3, 0, 0, 0]), src=ints([0, 3]), dst=ints([4, 6]))

    def calls(k, v, table, **kw):
        f = bml_b200.page_fork(k, v, a["src"], a["dst"], a["lens"], a["owned"], table, a["shared"], a["free"], a["used"], **kw)
        r = bml_b200.page_free(a["keep"], f.lens, f.owned, table, 16, f.shared, a["free"], f.free_used, **kw)
        c = bml_b200.page_compact(k, v, r.owned, table, r.shared, **kw)
        return [f.lens, f.owned, f.shared, f.free_used, f.status, r.lens, r.owned, r.shared, r.free_pages, r.free_used, r.status,
                c.block_table, c.shared, c.free_pages, c.free_used, table, k, v]

    def fresh():
        return pools[0].clone(), pools[1].clone(), a["table"].clone()

    want = [x.clone() for x in calls(*fresh())]
    assert P._fast not in (None, P._Wrappers)
    st = torch.cuda.Stream()
    x = fresh()
    torch.cuda.synchronize()
    got = calls(*x, stream=st)
    st.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    x, start = fresh(), fresh()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = calls(*x)
    for _ in range(3):
        for y, z in zip(x, start):
            y.copy_(z)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, w) for p, w in zip(got, want))
    del g
    monkeypatch.setattr(P, "_fast", P._Wrappers)
    assert all(torch.equal(p, w) for p, w in zip(calls(*fresh()), want))


def test_batcher_shares_and_returns_pages(cuda):
    """Requests fork, decode apart, are rolled back and removed; the cache of each
    stays what it would be alone, and no page is lost or held twice."""
    import bml_b200
    rng = np.random.default_rng(7)
    layers, heads, kv, d = 2, 4, 2, 64
    b = bml_b200.PagedBatcher(layers, heads, kv, d, n_pages=60, page_size=16, max_positions=256, dtype=torch.bfloat16,
                              max_requests=8, rope=False)
    kept = {}

    def held():
        s = State([], 16)
        s.n, s.n_pages, s.page = 8, 60, 16
        s.table, s.owned, s.shared = b.table.cpu().numpy(), b.owned.tolist(), b.shared.cpu().numpy()
        s.free, s.used = b.free.cpu().numpy(), int(b.used)
        s.check()
        for r in b.active:
            assert b.length(r) == kept[r][0].shape[1]
            for layer in range(layers):
                for x, y in zip(b.cache(r, layer), kept[r]):
                    assert torch.equal(x, y[layer])

    def step(new):
        b.begin(new)
        rows = [r for r in b.active if r in new]
        n = sum(new.values())
        xs = [(torch.randn(n, kv, d, device="cuda").bfloat16(), torch.randn(n, kv, d, device="cuda").bfloat16()) for _ in range(layers)]
        for layer, (k, v) in enumerate(xs):
            b.step(layer, torch.randn(n, heads, d, device="cuda").bfloat16(), k, v)
        at = 0
        for r in rows:
            t = new[r]
            kept[r] = tuple(torch.cat([kept[r][i], torch.stack([x[i][at:at + t] for x in xs])], 1) for i in range(2))
            at += t
        b.commit()

    prompt = [torch.randn(layers, 41, kv, d, device="cuda").bfloat16() for _ in "kv"]
    b.add("a", *prompt)
    kept["a"] = tuple(prompt)
    b.fork("a", ["b", "c"])
    kept["b"] = kept["c"] = kept["a"]
    held()
    assert int(b.used) == 5 and int(b.shared.sum()) == 4  # 3 pages, and a part-filled one each
    with pytest.raises(KeyError):
        b.fork("a", ["x", "b"])
    with pytest.raises(KeyError):
        b.fork("a", ["x", "x"])
    with pytest.raises(bml_b200.AtCapacity):
        b.fork("a", list(range(6)))
    for i in range(6):
        step({r: int(rng.integers(1, 20)) for r in b.active})
        held()
        if i == 1:
            b.fork("b", "d")
            kept["d"] = kept["b"]
            b.truncate("c", 40)
            kept["c"] = tuple(x[:, :40] for x in kept["c"])
        if i == 2:
            b.remove("a")
            del kept["a"]
            used = b.compact()
            assert used is b.used
        if i == 4:
            with pytest.raises(bml_b200.PageRefused):
                b.truncate("d", 17)      # inside a page that b holds too
            b.truncate("d", 16)
            kept["d"] = tuple(x[:, :16] for x in kept["d"])
        held()
    for r in list(b.active):
        b.remove(r)
        del kept[r]
        held()
    assert int(b.used) == 0 and int(b.shared.abs().sum()) == 0
    # a fork that finds no page admits nobody
    b.add("p")
    b2 = bml_b200.PagedBatcher(1, 4, 2, 64, n_pages=3, page_size=16, max_positions=64, max_requests=4)
    x = torch.zeros(1, 37, 2, 64, device="cuda", dtype=torch.bfloat16)
    b2.add("a", x, x)
    with pytest.raises(bml_b200.OutOfPages):
        b2.fork("a", "b")
    assert b2.active == ["a"] and int(b2.used) == 3 and int(b2.shared.sum()) == 0
    b2.begin({"a": 1})
    for call in (lambda: b2.fork("a", "b"), lambda: b2.truncate("a", 3), lambda: b2.remove("a"), lambda: b2.compact()):
        with pytest.raises(RuntimeError):
            call()
    b2.commit()
    with pytest.raises(ValueError):
        b2.truncate("a", -1)


@pytest.mark.parametrize("n,page,per,spare", [(600, 16, 60, 0), (4096, 16, 12, 5), (1, 16, 20000, 30), (64, 16, 6000, 200000)])
def test_free_of_a_long_list(cuda, n, page, per, spare):
    """The form over all SMs: short and long tiles of the list, one request and many."""
    rng = np.random.default_rng(n)
    s = State([int(x) for x in rng.integers(per * page // 2, per * page, n)], page, spare=spare, seed=n, share=n < 1000)
    for step in range(3):
        keep = [int(rng.choice([-1, 0, a, a // 2, a // 2 // page * page, a + 100])) for a in s.lens]
        p = call_free(s, keep)
        want = want_free(s, keep)
        for got, w in zip((p.lens, p.owned, p.shared, p.free_pages), want):
            assert (got.cpu().numpy() == np.asarray(w)).all()
        assert p.free_used.tolist() == [want[4]] and p.status.tolist() == want[5]
        s.lens, s.owned, s.shared, s.free, s.used = want[0], want[1], want[2], want[3], want[4]


@pytest.mark.parametrize("n_pages,n_free", [(20000, 7), (8, 20007), (20000, 0)])
def test_free_of_long_state_that_does_not_hold_together(cuda, n_pages, n_free):
    import bml_b200
    big = 0x7fffffff
    free = (([1, -7, big, 5, 5, 0, 2] * (n_free // 7 + 1))[:n_free]) if n_free else []
    p = bml_b200.page_free(ints([0, 0, 0, 5, -1]), ints([100, -5, 20, 30, 40]), ints([9, 2, -3, big, 2]),
                           ints([[5, -1, big, 5, 5, 7, 0, 0, 9]] * 5), 16, ints(([0, 3, -4] + [0] * n_pages)[:n_pages]),
                           ints(free), ints([big]))
    assert p.lens.tolist() == [0, -5, 20, 30, 40] and p.owned.tolist() == [0, 2, -3, big, 2]
    assert p.shared.tolist() == [0, 3] + [0] * (n_pages - 2)
    assert p.free_pages.tolist() == [x for x in free if x not in (5, 0)] + [x for x in free if x in (5, 0)]
    assert p.free_used.tolist() == [len([x for x in free if x not in (5, 0)])]


@pytest.mark.parametrize("n_pages,n,max_pages,held", [
    (8192, 16, 1024, 8192), (8192, 16, 1024, 5000), (8193, 16, 1024, 5000), (8192, 17, 1024, 4096), (8160, 2, 8192, 1),
    (33, 4096, 4, 20), (1, 1, 1, 1), (31, 1, 31, 31)])
def test_compact_at_the_edges_of_its_forms(cuda, n_pages, n, max_pages, held):
    import bml_b200
    rng = np.random.default_rng(held)
    order = rng.permutation(n_pages)[:held]
    table = np.full((n, max_pages), n_pages)
    owned = [held // n + (i < held % n) for i in range(n)]
    at = 0
    for i, k in enumerate(owned):
        table[i, :k] = order[at:at + k]
        at += k
    pools = [torch.arange(n_pages, device="cuda", dtype=torch.float16)[None, :, None, None, None].repeat(2, 1, 16, 1, 8) for _ in "kv"]
    mark = pools[0][:, :, 0, 0, 0].clone()
    u = bml_b200.page_compact(*pools, ints(owned), ints(table), ints(np.arange(n_pages) % 7))
    new = u.block_table.cpu().numpy()
    low = np.sort(order)
    move = dict(zip(low[low >= held], np.setdiff1d(np.arange(held), low)))
    want = np.array([[move.get(x, x) for x in row] for row in table])
    assert (new == want).all() and u.free_used.tolist() == [held] and u.free_pages.tolist() == list(range(n_pages))
    shared = np.zeros(n_pages, int)
    shared[[move.get(x, x) for x in order]] = order % 7
    assert (u.shared.cpu().numpy() == shared).all()
    for a, b in move.items():
        mark[:, b] = mark[:, a]
    for p in pools:
        assert torch.equal(p, mark[:, :, None, None, None].expand_as(p))


@pytest.mark.parametrize("n_pages,n,max_pages,held", [(2048, 8, 1024, 2048), (2048, 8, 1024, 1100), (2049, 8, 1024, 1100),
                                                      (2048, 9, 1024, 1100), (2047, 1, 8192, 700)])
def test_compact_between_its_forms(cuda, n_pages, n, max_pages, held):
    test_compact_at_the_edges_of_its_forms(None, n_pages, n, max_pages, held)


def test_long_forms_at_once_and_replayed(cuda, monkeypatch):
    """page_free over all SMs and page_compact of a large pool: on two streams at once,
    in a replayed graph and through ctypes, the same bits."""
    import bml_b200.paged as P
    rng = np.random.default_rng(9)
    s = State([int(x) for x in rng.integers(100, 900, 700)], 16, spare=20000, seed=9)
    keep = ints([int(rng.choice([-1, 0, a // 2 // 16 * 16])) for a in s.lens])
    a = [keep, ints(s.lens), ints(s.owned), ints(s.table), 16, ints(s.shared), ints(s.free), ints([s.used])]
    pools = [torch.randn(1, s.n_pages, 16, 1, 2, device="cuda") for _ in "kv"]

    def both(k, v, **kw):
        r = P.page_free(*a, **kw)
        c = P.page_compact(k, v, r.owned, a[3], r.shared, **kw)
        return [r.lens, r.owned, r.shared, r.free_pages, r.free_used, r.status, c.block_table, c.shared, c.free_pages, c.free_used, k, v]

    def fresh():
        return [p.clone() for p in pools]

    want = both(*fresh())
    assert int(want[4]) < s.used < s.n_pages and int(want[9]) == int(want[4])
    xs, st = [fresh() for _ in range(8)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [both(*x, stream=st[i & 1]) for i, x in enumerate(xs)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for g in got for x, w in zip(g, want))
    x, start = fresh(), fresh()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = both(*x)
    for _ in range(3):
        for y, z in zip(x, start):
            y.copy_(z)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for y, w in zip(got, want))
    monkeypatch.setattr(P, "_fast", P._Wrappers)
    assert all(torch.equal(y, w) for y, w in zip(both(*fresh()), want))


def test_pools_past_32_bits(cuda):
    """Pages whose bytes lie 4 GiB and more behind the pools' start."""
    import bml_b200
    n_pages = 70001
    k, v = (torch.empty(2, n_pages, 16, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in "kv")   # 4.6 GB each
    src = torch.randn(2, 2, 16, 8, 128, device="cuda").bfloat16()
    for p, x in ((k, src), (v, -src)):
        p[:, n_pages - 1], p[:, 40000] = x[0], x[1]
    table = ints([[n_pages - 1, -1], [-1, -1]])
    f = bml_b200.page_fork(k, v, ints([0]), ints([1]), ints([9, 0]), ints([1, 0]), table, ints([0] * n_pages),
                           ints([n_pages - 1, n_pages - 2]), ints([1]))
    assert f.status.tolist() == [0] and table.tolist() == [[n_pages - 1, -1], [n_pages - 2, -1]]
    for p, x in ((k, src), (v, -src)):
        assert torch.equal(p[:, n_pages - 2, :9], x[0][:, :9])
    c = bml_b200.page_compact(k, v, ints([2, 1]), ints([[n_pages - 1, 40000], [n_pages - 2, 7]]), ints([0] * n_pages))
    assert c.block_table.tolist() == [[2, 0], [1, 7]] and c.free_used.tolist() == [3]
    for p, x in ((k, src), (v, -src)):
        assert torch.equal(p[:, 2], x[0]) and torch.equal(p[:, 0], x[1]) and torch.equal(p[:, 1, :9], x[0][:, :9])


def test_a_tuple_names_one_request(cuda):
    """A request's name may be anything that a dictionary takes, in fork as in add."""
    import bml_b200
    b = bml_b200.PagedBatcher(1, 4, 2, 64, n_pages=8, page_size=16, max_positions=64, max_requests=4, rope=False)
    x = torch.randn(1, 20, 2, 64, device="cuda").bfloat16()
    b.add(("user", 1), x, x)
    b.fork(("user", 1), ("user", 2))
    assert b.active == [("user", 1), ("user", 2)]
    b.fork(("user", 2), [("user", 3), "c"])
    assert b.active == [("user", 1), ("user", 2), ("user", 3), "c"]
    for rid in b.active:
        assert all(torch.equal(y, x[0]) for y in b.cache(rid, 0))
    with pytest.raises(KeyError):
        b.fork("c", ("user", 1))
