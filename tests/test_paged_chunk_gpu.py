"""GPU tests of chunk_attention against its formula in 64 bits, with the cases and
tolerances of test_paged_gpu.py (the arithmetic is tree_attention's)."""
import ctypes as C

import numpy as np
import pytest
import torch

from test_paged_gpu import DT, TYPES, Paged, chain, check, ints, tol
from test_paged_masked_gpu import put, widen
from test_paged_stall_gpu import CODE

pytestmark = pytest.mark.gpu


def attend(c, **kw):
    import bml_b200
    return bml_b200.chunk_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, **kw)


def sees_of(c):
    return [chain(t, p) for t, p in zip(c.nodes, c.lens)]


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", [(8, 2, 64, 16), (16, 4, 128, 64), (5, 1, 128, 128), (3, 3, 64, 32),
                                             (32, 4, 64, 256), (24, 2, 128, 16), (8, 1, 128, 1024)])
def test_shapes(cuda, qt, ct, heads, kv, d, page):
    """Fresh prompts and later chunks, single tokens and none, around every edge of
    a tile of positions and of a group of rows."""
    for lens, nodes in (([0, 700, 0, 129, 5], [300, 1, 1, 0, 257]), ([0, 128, 127, 1], [128, 128, 129, 127]),
                        ([1000, 0], [33, 513])):
        c = Paged(lens, nodes, heads, kv, d, page, qt, ct, seed=heads + d)
        check(c, attend(c), sees_of(c), qt)


@pytest.mark.parametrize("qt,ct", TYPES)
def test_many_requests(cuda, qt, ct):
    """A server's mixed batch: most decode, some bring chunks; the same bits from
    run to run, and rows behind the last request left as they were."""
    rng = np.random.default_rng(3)
    for n, most, long in ((90, 40, 500), (7, 700, 300), (200, 1, 1), (3, 900, 3000)):
        lens = [int(x) for x in rng.integers(0, long, n)]
        nodes = [int(rng.integers(1, most + 1)) if rng.random() < 0.3 else int(rng.integers(0, 2)) for _ in range(n)]
        nodes[0] = most
        c = Paged(lens, nodes, 8, 2, 64, 16, qt, ct, seed=n, spare_rows=5)
        out = torch.full_like(c.q, 7.0)
        got = attend(c, out=out)
        assert got is out and (got[sum(nodes):] == 7).all()
        check(c, got, sees_of(c), qt)
        assert torch.equal(got[:sum(nodes)], attend(c)[:sum(nodes)])


@pytest.mark.parametrize("qt,ct", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["tokens", "chunks", "both", "short"])
def test_many_tiles_and_segments(cuda, qt, ct, d, kind):
    """Each SM gets long runs of tiles of few rows, many short segments, or row
    groups of one and of two row tiles in turns, of odd and even tile counts."""
    rng = np.random.default_rng(["tokens", "chunks", "both", "short"].index(kind))
    n, long, sizes = {"tokens": (60, 4000, [1]), "chunks": (24, 1500, [200, 333, 65]), "both": (90, 1700, [1, 1, 40, 33, 64, 100, 130]),
                      "short": (400, 200, [1, 2, 70])}[kind]
    lens = [int(x) for x in rng.integers(0, long, n)]
    nodes = [int(rng.choice(sizes)) for _ in range(n)]
    c = Paged(lens, nodes, 16, 4, d, 32, qt, ct, seed=n + d)
    got = attend(c)
    check(c, got, sees_of(c), qt, only=range(0, n, 7 if kind == "short" else 3))
    for _ in range(3):
        assert torch.equal(attend(c), got)


@pytest.mark.parametrize("qt,ct,d", [("bf16", "bf16", 128), ("f16", "f16", 64), ("f32", "f32", 128), ("f32", "bf16", 64)])
def test_long(cuda, qt, ct, d):
    """One long request that many CTAs share, a long fresh prompt, and a single
    token behind many positions."""
    for lens, nodes in (([20000], [300]), ([0], [3000]), ([30000, 0], [1, 1030])):
        c = Paged(lens, nodes, 8, 2, d, 64, qt, ct, seed=5)
        check(c, attend(c), sees_of(c), qt)


@pytest.mark.parametrize("qt,ct", TYPES)
def test_as_tree_attention(cuda, qt, ct):
    """Up to 256 tokens a request both calls compute the same, within twice the
    tolerance of one; scales too, 0 among them."""
    import bml_b200
    c = Paged([300, 7, 0, 1000], [256, 3, 100, 1], 12, 4, 128, 32, qt, ct, seed=6)
    for scale in (-1.0, 0.0, 0.2, 1e-20):
        a, b = attend(c, scale=scale), bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, scale=scale)
        for i in range(4):
            s = slice(int(c.start[i]), int(c.start[i + 1]))
            want, ab, bm = c.want(i, chain(c.nodes[i], c.lens[i]), None if scale < 0 else scale)
            assert ((a[s].double() - want).abs() <= tol(qt, want, ab, bm)).all(), (scale, i)
            assert ((a[s].double() - b[s].double()).abs() <= 2 * tol(qt, want, ab, bm)).all()


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("heads,kv", [(130, 1), (256, 2), (300, 1), (127, 1)])
def test_many_heads_of_one(cuda, qt, ct, heads, kv):
    """Groups of about 128 q heads and of more than a row group holds."""
    c = Paged([40, 0, 300], [3, 270, 1], heads, kv, 64, 16, qt, ct, seed=7)
    check(c, attend(c), sees_of(c), qt)


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_refused_requests_and_bad_pages(cuda, qt, ct, d):
    """Requests that the plan refused (kv_len 0), with more positions than their
    table, or whose rows leave the token rows, are zero or left; pages outside the
    pool count as masked."""
    lens, nodes = [300, 50, 90, 100, 33], [5, 700, 4, 306, 3]
    c = Paged(lens, nodes, 8, 2, d, 16, qt, ct, seed=13, spare_rows=4)
    kv = c.kv_lens.clone()
    kv[0] = 0
    kv[1] = 699                          # fewer positions than new tokens
    kv[2] = c.table.shape[1] * 16 + 1
    c.table[3, 2] = c.k.shape[0]         # positions 32..47
    c.table[3, 4] = -5                   # 64..79
    c.table[3, 10] = 1 << 30             # 160..175, in the chunk
    c.kv_lens = kv
    out = torch.full_like(c.q, 7.0)
    got = attend(c, out=out)
    s = c.start.tolist()
    assert (got[:s[3]] == 0).all() and (got[s[5]:] == 7).all()
    see = chain(306, 100)
    see[:, 32:48] = see[:, 64:80] = see[:, 160:176] = False
    check(c, got, [None, None, None, see, chain(3, 33)], qt, only=[3, 4])
    c.table[4] = 1 << 30                 # all its pages are bad: it sees nothing
    assert (attend(c, out=out)[s[4]:s[5]] == 0).all()
    c.table[3, :] = -1                   # and one of several row groups
    assert (attend(c, out=out)[s[3]:s[5]] == 0).all()
    bad = c.start.clone()
    bad[5] = 1000                        # rows that leave the tokens are not written
    c.start = bad
    out.fill_(7.0)
    assert (attend(c, out=out)[s[4]:] == 7).all()


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 64), (2, 2, 128), (3, 1, 64)])
@pytest.mark.parametrize("start,rows", [([0, 300, 700], 600), ([0, 300, 310], 305), ([0, 300, 301], 300), ([0, 300, 200], 320),
                                        ([0, 300, 1 << 30], 513), ([0, 300, -7], 500), ([0, 300, 900, 340], 600),
                                        ([-3, 60, 360], 400), ([700, 100, 400], 700), ([0, 300, 650, 600, 900], 888)])
def test_neighbours_of_requests_whose_rows_are_none(cuda, qt, ct, heads, kv, d, start, rows):
    """A request whose rows leave the token rows, or that begins behind its end, is
    not served; the requests beside it are, each to its own end, and rows that no
    request holds stay as they were."""
    n = len(start) - 1
    good = [i for i in range(n) if 0 <= start[i] < start[i + 1] <= rows]
    nodes = [start[i + 1] - start[i] if i in good else 5 for i in range(n)]
    lens = [90, 20, 7, 500][:n]
    c = Paged(lens, nodes, heads, kv, d, 32, qt, ct, seed=rows, spare_rows=rows - sum(nodes))
    c.start = ints(start)
    out = torch.full_like(c.q, 7.0)
    got = attend(c, out=out)
    check(c, got, sees_of(c), qt, only=good)
    idle = torch.ones(rows, dtype=torch.bool)
    for i in good:
        idle[start[i]:start[i + 1]] = False
    assert (got[idle.cuda()] == 7).all()


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_later_tokens_do_not_reach_a_row(cuda, qt, ct, d):
    """NaN, infinities and the largest values in K and V of a chunk's later tokens,
    and in memory that nobody holds, leave the rows before them as they are; an
    infinity that a row sees makes its column infinite, NaN makes it NaN."""
    lens, nodes = [0, 203, 77], [400, 300, 1]
    inf, nan = float("inf"), float("nan")
    big = {"bf16": 3.38e38, "f16": 65504.0, "f32": 1e38}[ct]
    for i, at, k, v in ((0, 399, nan, inf), (0, 130, None, inf), (1, 299, inf, nan), (1, 255, nan, big), (0, 31, None, nan),
                        (1, 0, None, -inf)):
        c = Paged(lens, nodes, 8, 2, d, 16, qt, ct, seed=50 + d)
        put(c, i, lens[i] + at, 16, k=k, v=None)
        if v is not None:
            page = int(c.table[i, (lens[i] + at) // 16])
            c.v[page, (lens[i] + at) % 16, :, 5] = v
            c.vs[i][lens[i] + at, :, 5] = v
        got = attend(c)
        a = int(c.start[i])
        # rows that do not see it, by the formula without it
        kept, old = c.ks[i].clone(), c.vs[i].clone()
        c.ks[i][lens[i] + at] = 0
        c.vs[i][lens[i] + at] = 0
        see = chain(nodes[i], lens[i])
        see[at:, lens[i] + at] = False
        want, ab, bm = c.want(i, see)
        low = got[a:a + at].double()
        assert torch.isfinite(low).all()
        assert ((low - want[:at]).abs() <= tol(qt, want, ab, bm)[:at]).all()
        c.ks[i], c.vs[i] = kept, old
        high = got[a + at:a + nodes[i]].float()
        if k is None:
            col = high[:, :, 5]
            assert (torch.isnan(col) if v != v else torch.isposinf(col) if v > 0 else torch.isneginf(col)).all()
            rest = [x for x in range(d) if x != 5]
            assert torch.isfinite(high[:, :, rest]).all()
        check(c, got, sees_of(c), qt, only=[x for x in range(3) if x != i])


@pytest.mark.parametrize("qt,ct", TYPES)
def test_infinities_far_from_the_chunk(cuda, qt, ct):
    """In committed positions that every row sees, weightless ones among them."""
    inf = float("inf")
    c = Paged([2500, 40], [300, 20], 8, 2, 64, 16, qt, ct, seed=60)
    for pos, h, col, x in ((3, 0, 7, inf), (1300, 1, 8, -inf), (2499, 1, 60, inf), (130, 0, 9, inf), (900, 0, 9, -inf)):
        page = int(c.table[0, pos // 16])
        c.v[page, pos % 16, h, col] = x
    c.q[:, :4].abs_()
    page = int(c.table[0, 0])
    c.k[page, 3, 0] = -50.0                 # weight 0 in 32 bits, and an infinite value
    c.ks[0][3, 0] = -50.0
    got = attend(c)[:300]
    assert torch.isposinf(got[:, :4, 7]).all() and torch.isneginf(got[:, 4:, 8]).all() and torch.isposinf(got[:, 4:, 60]).all()
    assert torch.isnan(got[:, :4, 9]).all()
    got[:, :4, 7] = got[:, 4:, 8] = got[:, 4:, 60] = got[:, :4, 9] = 0
    want, ab, bm = c.want(0, chain(300, 2500))
    want[:, :4, 7] = want[:, 4:, 8] = want[:, 4:, 60] = want[:, :4, 9] = 0
    assert ((got.double() - want).abs() <= tol(qt, want, ab, bm)).all()


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("n,total", [(1, 128), (1, 129), (8, 64), (8, 65), (9, 64), (1, 256), (1, 257), (30, 256), (30, 257), (1024, 200),
                                     (1025, 200)])
def test_between_the_forms_for_few_tokens(cuda, qt, ct, n, total):
    """Around the sizes where another kernel takes the call: idle requests, a wide
    one, a refused one; rows behind the last request's stay as they were."""
    rng = np.random.default_rng(n + total)
    nodes = [0] * n
    for i in rng.integers(0, n, total // 2) if n > 1 else []:
        nodes[int(i)] += 1
    nodes[n // 2] += total - sum(nodes)
    c = Paged([int(x) for x in rng.integers(0, 30 if n > 100 else 700, n)], nodes, 8, 2, 64 if n % 2 else 128, 16, qt, ct, seed=n,
              spare_rows=3)
    bad = int(np.argmax([0 if i == n // 2 else x for i, x in enumerate(nodes)])) if n > 1 else -1
    if bad >= 0:
        c.kv_lens[bad] = 0
    out = torch.full_like(c.q, 7.0)
    got = attend(c, out=out)
    assert got is out and (out[total:] == 7.0).all()
    check(c, got, sees_of(c), qt, only=[i for i in range(n) if i != bad][::1 if n < 100 else 9] + [n // 2])
    if bad >= 0:
        assert (got[int(c.start[bad]):int(c.start[bad]) + nodes[bad]] == 0).all()


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("nodes", [[0] * 40 + [400], [1] * 30 + [90], [0] * 60 + [70, 1]])
def test_what_the_caller_says_of_the_batch(cuda, qt, ct, nodes):
    """n_live and max_new, right or wrong, change the kernel and not the result."""
    c = Paged([300] * (len(nodes) - 1) + [900], nodes, 8, 2, 128, 32, qt, ct, seed=71)
    for live, most in ((0, 0), (sum(x > 0 for x in nodes), max(nodes)), (1, 1), (len(nodes) + 5, 0), (2, 1 << 30), (1, 0)):
        for kw in ({}, {"out": torch.empty_like(c.q)}):
            check(c, attend(c, n_live=live, max_new=most, **kw), sees_of(c), qt)
    for bad in ({"n_live": -1}, {"max_new": 1 << 31}):
        with pytest.raises(ValueError):
            attend(c, **bad)


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nodes", [[300, 5], [60, 40], [1, 3]])
def test_keys_of_minus_infinite_scores(cuda, qt, ct, d, nodes):
    """An infinite key whose scores are -inf has weight 0 (and no lower term of a split
    operand makes NaN of it); one whose scores are +inf makes its rows NaN."""
    inf = float("inf")
    c = Paged([700, 90], nodes, 8, 2, d, 32, qt, ct, seed=61)
    c.q[:, :, 3] = -c.q[:, :, 3].abs() - 0.4
    places = ((0, 17), (0, 640), (1, 89))
    for i, pos in places:
        c.k[int(c.table[i, pos // 32]), pos % 32, :, 3] = inf
        c.ks[i][pos, :, 3] = 0
    got = attend(c)
    for i in range(2):
        see = chain(nodes[i], c.lens[i])
        for j, pos in places:
            if i == j:
                see[:, pos] = False
        want, ab, bm = c.want(i, see)
        have = got[int(c.start[i]):int(c.start[i]) + nodes[i]].double()
        assert torch.isfinite(have).all() and ((have - want).abs() <= tol(qt, want, ab, bm)).all()
    c.k[int(c.table[0, 0]), 17, 0, 3] = -inf      # scores of the first kv head's rows
    got = attend(c)[:nodes[0]]
    assert torch.isnan(got[:, :4]).all() and torch.isfinite(got[:, 4:]).all()


def test_offsets_past_32_bits(cuda):
    """Pages at the end of a pool of more than 2^31 elements (4.5 GB)."""
    c = Paged([200, 31], [290, 1], 8, 8, 128, 64, "bf16", "bf16", seed=14)
    n_pages = (1 << 31) // (64 * 8 * 128) + 40
    want, want32 = attend(c), None
    q32 = c.q.float()
    small = (c.k, c.v, c.table)
    k = torch.empty(n_pages, 64, 8, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    used = c.k.shape[0]
    k[-used:], v[-used:] = c.k, c.v
    c.k, c.v, c.table = k, v, torch.where(c.table >= 0, c.table + (n_pages - used), c.table).int()
    assert torch.equal(attend(c), want)
    c.q = q32
    got32 = attend(c)
    c.k, c.v, c.table = small
    want32 = attend(c)
    assert torch.equal(got32, want32)
    check(c, want32, sees_of(c), "f32")


def test_more_pieces_than_one_launch(cuda):
    """32-bit queries over more requests than the kernels take at once, and a chunk
    of more pieces than that."""
    lens = [i % 37 for i in range(1500)]
    c = Paged(lens, [1] * 1500, 4, 2, 64, 16, "f32", "bf16", seed=15)
    check(c, attend(c), sees_of(c), "f32", only=[0, 1, 700, 1023, 1024, 1025, 1499])
    c = Paged([5], [2200], 256, 1, 64, 64, "f32", "f16", seed=16)
    got = attend(c)
    rows = [0, 1, 1000, 1023, 1024, 1025, 2047, 2048, 2199]
    k, v = c.ks[0][:, 0].double(), c.vs[0][:, 0].double()
    for t in rows:
        n = 6 + t
        s = c.q[t].double() @ k[:n].T / 8
        p = torch.softmax(s, -1)
        b = (c.q[t].double().abs() @ k[:n].abs().T / 8).amax(-1, keepdim=True)
        assert ((got[t].double() - p @ v[:n]).abs() <= tol("f32", None, p @ v[:n].abs(), b)).all()


@pytest.mark.parametrize("qt,ct,d", [("bf16", "bf16", 128), ("f16", "f16", 64), ("f32", "f32", 64), ("f32", "f16", 128)])
def test_streams_and_graphs(cuda, qt, ct, d):
    """Another stream; two graphs whose replays overlap on two streams, each behind
    its own writes of the lengths; new lengths in the same graph."""
    cs = [Paged([3000, 10, 77], [8, 300, 1], 8, 2, d, 64, qt, ct, seed=s) for s in (20, 21)]
    want = [attend(c) for c in cs]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = attend(cs[0], stream=s)
    s.synchronize()
    assert torch.equal(got, want[0])
    graphs, outs, full = [], [], [c.kv_lens.clone() for c in cs]
    for c, f in zip(cs, full):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.kv_lens.zero_()
            attend(c)
            c.kv_lens.copy_(f)
            outs.append(attend(c))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    full[0].copy_(ints([2500, 305, 60]))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], attend(cs[0]))
    del graphs


def test_workspace_of_the_callers(cuda):
    import bml_b200
    c = Paged([300, 5], [290, 3], 8, 2, 64, 16, "bf16", "bf16", seed=22)
    n = bml_b200.chunk_workspace_size(64, c.q.shape[0], 2)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    want = attend(c)
    assert torch.equal(attend(c, workspace=ws), want)
    with pytest.raises(bml_b200.BmlInvalid):
        attend(c, workspace=ws[:n - 4])
    c.q = c.q.float()
    assert torch.equal(attend(c, workspace=ws), attend(c))


def test_both_ways_agree_and_refusals(cuda, monkeypatch):
    import bml_b200
    import bml_b200.paged as P
    c = Paged([40, 3], [300, 1], 4, 2, 64, 16, "bf16", "bf16", seed=30)
    want = attend(c, scale=0.3)
    assert P._fast not in (None, P._Wrappers)
    good = [c.q, c.k, c.v, c.table, c.kv_lens, c.start]
    for way in (P._fast, P._Wrappers):
        monkeypatch.setattr(P, "_fast", way)
        assert torch.equal(attend(c, scale=0.3), want)
        for i, x, err in ((0, c.q.double(), TypeError), (0, c.q.half(), bml_b200.BmlUnsupported), (0, c.q.cpu(), ValueError),
                          (0, c.q[:, :3].contiguous(), bml_b200.BmlInvalid), (0, c.q.transpose(0, 1), ValueError),
                          (0, torch.cat([c.q, c.q], 2), ValueError), (1, c.k.float(), TypeError), (2, c.v[:1], ValueError),
                          (3, c.table.long(), TypeError), (3, c.table[:1], ValueError), (4, c.kv_lens[:1], ValueError),
                          (5, c.start[:2], ValueError), (5, c.start.long(), TypeError)):
            args = list(good)
            args[i] = x
            with pytest.raises(err):
                bml_b200.chunk_attention(*args)
        with pytest.raises(bml_b200.BmlInvalid):
            attend(c, scale=float("nan"))
        with pytest.raises(bml_b200.BmlInvalid):
            attend(c, out=c.q)
        assert bml_b200.chunk_attention(c.q[:0], *good[1:5], c.start * 0).shape == (0, 4, 64)


@pytest.mark.parametrize("qt,ct,heads,nodes,d", [("bf16", "bf16", 16, [20, 300], 128), ("f16", "f16", 16, [1, 1], 64),
                                                 ("f16", "f16", 8, [700, 600], 64), ("f32", "f32", 16, [40, 300], 128)])
def test_stalled_copies_leave_nan(cuda, qt, ct, heads, nodes, d):
    """Copies that never come end the launch by themselves after a short limit and
    leave NaN in every row, and the next call is right."""
    import bml_b200
    import bml_b200._lib as L
    lens = [(37 * i) % 300 for i in range(60)]
    c = Paged(lens, nodes * 30, heads, 4, d, 16, qt, ct, seed=70)
    widen(c, 16, 4096)
    n, page, kv, _ = c.k.shape
    size = bml_b200.chunk_workspace_size(d, c.q.shape[0], 60)

    def stalled(flags):
        out, ws = torch.full_like(c.q, 7.0), torch.full((size // 4,), 0.5, device="cuda")
        a = [t.data_ptr() for t in (c.q, c.k, c.v, c.table, c.kv_lens, c.start, out, ws)]
        st = L.lib().bml_diag_attn_chunk(a[0], CODE[qt], c.q.shape[0], heads, kv, d, a[1], a[2], CODE[ct], n, page, a[3],
                                         c.table.shape[1], a[4], a[5], 60, -1.0, a[6], a[7], ws.numel() * 4, 20_000_000, flags,
                                         C.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert st == 0, L.last_error()
        torch.cuda.synchronize()
        return out

    assert torch.isnan(stalled(L.BML_DIAG_STALL)).all()
    out = stalled(0)
    assert torch.equal(out, attend(c))
    check(c, out, sees_of(c), qt, only=[0, 1, 33, 59])


@pytest.mark.parametrize("ct,d", [("bf16", 128), ("f16", 64)])
def test_stalled_copies_of_16_bit_pages_under_32_bit_queries(cuda, ct, d):
    test_stalled_copies_leave_nan(None, "f32", ct, 16, [40, 300], d)


@pytest.mark.parametrize("qt,ct", [("bf16", "bf16"), ("f32", "f16")])
def test_batcher_takes_prompts_in_chunks(cuda, qt, ct):
    """A prompt that comes in chunks beside decoding requests: rows in the cache and
    every step's attention."""
    import bml_b200
    layers, heads, kv, d = 2, 8, 2, 64
    b = bml_b200.PagedBatcher(layers, heads, kv, d, n_pages=120, page_size=16, max_positions=1024, dtype=DT[ct], max_requests=4,
                              rope=False)
    kept = {}
    for r in "abc":
        b.add(r)
        kept[r] = tuple(torch.zeros(layers, 0, kv, d, device="cuda", dtype=DT[ct]) for _ in "kv")
    with pytest.raises(ValueError):
        b.begin({"a": [-1, 0]}, chunks=True)
    with pytest.raises(ValueError):
        b.begin({"a": 300})
    for new in ({"a": 300, "b": 1}, {"a": 401, "b": 1, "c": 257}, {"a": 1, "c": 3}, {"b": 30}):
        b.begin(new, chunks=True)
        n = sum(new.values())
        for layer in range(layers):
            q = torch.randn(n, heads, d, device="cuda").to(DT[qt])
            k, v = (torch.randn(n, kv, d, device="cuda").to(DT[ct]).to(DT[qt]) for _ in "kv")
            out = b.step(layer, q, k, v)
            at = 0
            for r in b.active:
                t = new.get(r, 0)
                if not t:
                    continue
                p = b.length(r)
                case = object.__new__(Paged)
                old = [x[layer] for x in kept[r]] if layer else [x[layer, :p] for x in kept[r]]
                case.ks, case.vs = [torch.cat([old[0][:p], k[at:at + t].to(DT[ct])])], [torch.cat([old[1][:p], v[at:at + t].to(DT[ct])])]
                case.q, case.start, case.nodes, case.lens, case.group = q[at:at + t], [0], [t], [p], heads // kv
                check(case, out[at:at + t], [chain(t, p)], qt)
                if layer == 0:
                    kept[r] = tuple(torch.cat([x, torch.zeros(layers, t, kv, d, device="cuda", dtype=DT[ct])], 1) for x in kept[r])
                for x, y in zip(kept[r], (k, v)):
                    x[layer, p:p + t] = y[at:at + t].to(DT[ct])
                at += t
        b.commit()
        for r in b.active:
            for layer in range(layers):
                for x, y in zip(b.cache(r, layer), kept[r]):
                    assert torch.equal(x, y[layer])
    b.begin({"a": 300}, chunks=True)
    with pytest.raises(ValueError):
        b.verify(torch.zeros(300, 4, device="cuda"), None, ints([0] * 300), torch.zeros(300, device="cuda"), torch.zeros(4, device="cuda"))


def test_a_serving_run(cuda):
    """The calls as a server makes them: a prompt in chunks, forked, its drafts
    verified on the GPU, one sample rolled back, requests ended and the pool packed,
    against commit() with the same paths on a batcher that shares nothing."""
    import bml_b200
    layers, heads, kv, d, vocab = 2, 8, 2, 64, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    made = [bml_b200.PagedBatcher(layers, heads, kv, d, n_pages=90, page_size=16, max_positions=512, max_requests=4) for _ in "ab"]
    share, alone = made

    def step(rows, new, **kw):
        n = sum(x if isinstance(x, int) else len(x) for x in new.values())
        xs = [(rnd(n, heads, d), rnd(n, kv, d), rnd(n, kv, d)) for _ in range(layers)]
        outs = []
        for b, r in zip(made, rows):
            b.begin({r[k]: x for k, x in new.items()}, **kw)
            outs.append([b.step(i, q.clone(), k.clone(), v) for i, (q, k, v) in enumerate(xs)])
        for x, y in zip(*outs):
            assert torch.equal(x, y)

    # the same prompt once, and into each request that does not share it
    n = 300
    share.add("p0")
    for i in range(3):
        alone.add(f"p{i}")
    xs = [(rnd(n, heads, d), rnd(n, kv, d), rnd(n, kv, d)) for _ in range(layers)]
    share.begin({"p0": n}, chunks=True)
    first = [share.step(i, q.clone(), k.clone(), v) for i, (q, k, v) in enumerate(xs)]
    share.commit()
    for r in range(3):
        alone.begin({f"p{r}": n}, chunks=True)
        for i, (q, k, v) in enumerate(xs):
            assert torch.equal(alone.step(i, q.clone(), k.clone(), v), first[i])
        alone.commit()
    share.fork("p0", ["p1", "p2"])
    assert int(share.used) < int(alone.used)
    same = {f"p{r}": f"p{r}" for r in range(3)}
    for it in range(3):
        trees = {f"p{r}": [-1, 0, 0, 1, 1, 2][:3 + r + it % 2] for r in range(3)}
        step([same, same], trees)
        n = sum(len(x) for x in trees.values())
        p = torch.softmax(torch.randn(n, vocab, device="cuda", generator=g), -1)
        q = torch.softmax(p.log() + 0.3 * torch.randn(n, vocab, device="cuda", generator=g), -1)
        tok = torch.randint(0, vocab, (n,), device="cuda", generator=g, dtype=torch.int32)
        u, un = torch.rand(n, device="cuda", generator=g), torch.rand(4, device="cuda", generator=g)
        path, count, token = share.verify(p, q, tok, u, un)
        paths = {r: path[share.place(r)][:int(count[share.place(r)])].tolist() for r in trees}
        alone.commit(paths)
        if it == 0:
            for b in made:
                b.truncate("p1", 300)
            share.compact()
        if it == 1:
            for b in made:
                b.remove("p0")
            same.pop("p0")
            share.fork("p2", "p0")
            alone.add("p0", *(torch.stack([alone.cache("p2", i)[w] for i in range(layers)]) for w in range(2)))
            same["p0"] = "p0"
            share.compact()
        for r in share.active:
            assert share.length(r) == alone.length(r)
            for layer in range(layers):
                for x, y in zip(share.cache(r, layer), alone.cache(r, layer)):
                    assert torch.equal(x, y)
    for b in made:
        for r in list(b.active):
            b.remove(r)
        assert int(b.used) == 0 and int(b.shared.abs().sum()) == 0
