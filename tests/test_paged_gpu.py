"""GPU tests of the paged cache: page_plan against a plain Python planner,
paged_append and tree_attention against their formulas in 64 bits,
paged_commit against moves one row at a time, and the four together through
PagedBatcher.

Tolerances of the attention, per output element, from its arithmetic, with
A = sum p |v| and B = max over positions of sum |q_i k_i| * scale:
* 16-bit: the softmax weights are rounded to the type (half a step,
  eps / 2 each, so eps / 2 * A in the sum), the output once more
  (eps / 2 * |out|); the exponential is good to 1e-4 (a fitted cubic, 7.7e-5)
  and scores are f32 sums of exact products: B * 64 * 2^-23 covers their
  rounding, which moves a weight by as much relatively.
* 32-bit: a TF32 split leaves 3 * 2^-22 of each product, its sums at most 64
  roundings of 2^-23: B * (3 * 2^-22 + 64 * 2^-23) on a weight, plus
  2^-18 for the exponential and the sums over positions."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def starts_of(nodes):
    return torch.tensor(np.concatenate([[0], np.cumsum(nodes)]), dtype=torch.int32, device="cuda")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def random_parents(rng, t):
    return [int(max(-1, j - 1 - rng.integers(0, 4))) for j in range(t)]


def mask_of(parents):
    """Rows of bools: node j sees node a."""
    t = len(parents)
    m = np.zeros((t, t), bool)
    for j, a in enumerate(parents):
        if a >= 0:
            m[j] |= m[a]
        m[j, j] = True
    return m


def pack(masks, words):
    out = np.zeros((sum(len(m) for m in masks), words), np.uint64)
    r = 0
    for m in masks:
        for j in range(len(m)):
            for a in np.flatnonzero(m[j]):
                out[r, a // 64] |= np.uint64(1) << np.uint64(a % 64)
            r += 1
    return torch.from_numpy(out.view(np.int64)).cuda()


class Paged:
    """Requests of `lens` committed positions and `nodes` new ones on shuffled
    pages; everything that no request holds is NaN."""

    def __init__(self, lens, nodes, heads, kv, d, page, q, cache, seed=0, spare_rows=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rng = np.random.default_rng(seed)
        total = [a + b for a, b in zip(lens, nodes)]
        need = [-(-t // page) for t in total]
        n_pages = sum(need) + 2
        order = rng.permutation(n_pages)
        mp = max(need + [1]) + 1
        table = np.full((len(lens), mp), -1, np.int64)
        self.k = torch.full((n_pages, page, kv, d), float("nan"), device="cuda", dtype=DT[cache])
        self.v = self.k.clone()
        at = 0
        self.ks, self.vs = [], []
        for i, (t, c) in enumerate(zip(total, need)):
            pages = order[at:at + c]
            table[i, :c] = pages
            at += c
            k = torch.randn(t, kv, d, device="cuda", generator=g).to(DT[cache])
            v = torch.randn(t, kv, d, device="cuda", generator=g).to(DT[cache])
            pos = torch.arange(t, device="cuda")
            pg = torch.from_numpy(pages).cuda()
            if t:
                self.k[pg[pos // page], pos % page] = k
                self.v[pg[pos // page], pos % page] = v
            self.ks.append(k)
            self.vs.append(v)
        self.table = ints(table)
        self.q = torch.randn(sum(nodes) + spare_rows, heads, d, device="cuda", generator=g).to(DT[q])
        self.kv_lens = ints(total)
        self.start = starts_of(nodes)
        self.lens, self.nodes, self.group = lens, nodes, heads // kv

    def want(self, i, sees, scale=None):
        """(out, sum p|v|, max score sum) of request i, f64; sees: bools [T, L]."""
        k, v = self.ks[i].double(), self.vs[i].double()
        a = int(self.start[i])
        q = self.q[a:a + self.nodes[i]].double()
        sc = (1.0 / q.shape[2] ** 0.5) if scale is None else scale
        kk = k.repeat_interleave(self.group, 1)
        vv = v.repeat_interleave(self.group, 1)
        s = torch.einsum("thd,lhd->htl", q, kk) * sc
        bmax = (torch.einsum("thd,lhd->htl", q.abs(), kk.abs()) * abs(sc)).nan_to_num(0, 0, 0).amax(-1)
        see = torch.as_tensor(sees, device="cuda")[None]
        p = torch.softmax(s.masked_fill(~see, float("-inf")), -1).masked_fill(~see, 0.0)
        p = torch.where(see.any(-1, keepdim=True), p, torch.zeros_like(p))
        vz = torch.where(torch.as_tensor(sees, device="cuda").any(0)[:, None, None], vv, torch.zeros_like(vv))
        return (torch.einsum("htl,lhd->thd", p, vz), torch.einsum("htl,lhd->thd", p, vz.abs()), bmax.T[..., None])


def chain(t, p):
    return np.concatenate([np.ones((t, p), bool), np.tril(np.ones((t, t), bool))], 1)


def tol(qt, out, a, b):
    if qt == "f32":
        return (b * (3 * 2.0 ** -22 + 64 * 2.0 ** -23) + 2.0 ** -18) * a + 1e-30
    e = torch.finfo(DT[qt]).eps / 2
    return (e + 1e-4 + b * 64 * 2.0 ** -23) * a + e * out.abs() + torch.finfo(DT[qt]).tiny


def check(c, got, sees, qt, scale=None, only=None):
    for i in range(len(c.lens)) if only is None else only:
        a = int(c.start[i])
        if c.nodes[i] == 0:
            continue
        want, ab, b = c.want(i, sees[i], scale)
        have = got[a:a + c.nodes[i]].double()
        assert torch.isfinite(have).all(), f"request {i}"
        over = ((have - want).abs() - tol(qt, want, ab, b)).max().item()
        assert over <= 0, (i, c.lens[i], c.nodes[i], over, (have - want).abs().max().item())


TYPES = [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f32", "f16")]


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("heads,kv,d,page", [(8, 2, 64, 16), (16, 4, 128, 64), (5, 1, 128, 128), (3, 3, 64, 32),
                                             (32, 4, 64, 256), (24, 2, 128, 16)])
def test_tree_matches_f64(cuda, qt, ct, heads, kv, d, page):
    import bml_b200
    rng = np.random.default_rng(heads + d)
    lens = [0, 0, 1, 15, 16, 127, 128, 113, 300, 1025, 700, 40]
    nodes = [1, 9, 1, 2, 17, 1, 5, 15, 0, 33, 64, 61]
    c = Paged(lens, nodes, heads, kv, d, page, qt, ct, seed=d + page)
    masks = [mask_of(random_parents(rng, t)) for t in nodes]
    sees = [np.concatenate([np.ones((t, p), bool), m.reshape(t, t)], 1) for t, p, m in zip(nodes, lens, masks)]
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, mask=pack(masks, 1))
    check(c, got, sees, qt)


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 64), (8, 2, 128)])
def test_wide_drafts(cuda, qt, ct, heads, kv, d):
    """Drafts of up to 256 nodes (2 to 4 mask words, several row groups)."""
    import bml_b200
    rng = np.random.default_rng(3)
    for words, nodes in ((2, [65, 128, 3]), (4, [256, 129, 1, 200])):
        lens = [77, 500, 0, 1111][:len(nodes)]
        c = Paged(lens, nodes, heads, kv, d, 32, qt, ct, seed=words)
        masks = [mask_of(random_parents(rng, t)) for t in nodes]
        sees = [np.concatenate([np.ones((t, p), bool), m], 1) for t, p, m in zip(nodes, lens, masks)]
        got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, mask=pack(masks, words))
        check(c, got, sees, qt)


@pytest.mark.parametrize("qt,ct", TYPES)
def test_chain_and_decode(cuda, qt, ct):
    """No mask: chains, and T = 1, which is decode_batched over pages."""
    import bml_b200
    lens, nodes = [3, 0, 260, 1000, 64], [4, 256, 1, 40, 0]
    c = Paged(lens, nodes, 8, 2, 128, 16, qt, ct, seed=5)
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, scale=0.11)
    check(c, got, [chain(t, p) for t, p in zip(nodes, lens)], qt, scale=0.11)
    lens = [0, 1, 127, 128, 129, 2000, 511]
    c = Paged(lens, [1] * len(lens), 32, 4, 64, 64, qt, ct, seed=6)
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start)
    check(c, got, [chain(1, p) for p in lens], qt)
    if qt == "f32":
        old = bml_b200.decode_batched(c.q, c.ks, c.vs)
        assert (old - got).abs().max().item() < 1e-4  # decode's own tolerance


@pytest.mark.parametrize("qt,ct", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")])
def test_many_requests_and_long(cuda, qt, ct):
    """A batch that cuts units at many places, and one long request that many
    CTAs share; the same bits from run to run."""
    import bml_b200
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(0, 900, 70)] + [40000]
    nodes = [int(x) for x in rng.integers(0, 20, 70)] + [23]
    c = Paged(lens, nodes, 8, 2, 64, 16, qt, ct, seed=9)
    masks = [mask_of(random_parents(rng, t)) for t in nodes]
    sees = [np.concatenate([np.ones((t, p), bool), m.reshape(t, t)], 1) for t, p, m in zip(nodes, lens, masks)]
    m = pack(masks, 1)
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, mask=m)
    check(c, got, sees, qt)
    again = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, mask=m)
    assert torch.equal(got, again)


@pytest.mark.parametrize("qt,ct", TYPES)
def test_masked_places_do_not_reach_a_row(cuda, qt, ct):
    """Rows whose mask leaves nothing are zero; NaN and infinities in K and V
    of nodes that a row does not see leave it as it is, and those of a node
    that it sees reach it; masks may skip a node itself."""
    import bml_b200
    lens, nodes = [0, 200, 0], [6, 7, 70]
    c = Paged(lens, nodes, 8, 2, 64, 16, qt, ct, seed=12)
    rng = np.random.default_rng(1)
    masks = [np.zeros((6, 6), bool), np.zeros((7, 7), bool), rng.random((70, 70)) < 0.3]
    masks[0][1, 0] = masks[0][2, 5] = masks[0][5, 5] = True   # rows 0, 3, 4 see nothing
    masks[1][0, 1] = masks[1][6, 2] = masks[1][6, 6] = True
    masks[2][:, 67:] = False
    masks[2][69, 68] = True                                    # node 68 (an infinity) is seen by row 69 only
    masks[2][:, 3] = False                                     # node 3 (NaN) by nobody
    for i, node, k, v in ((0, 3, float("nan"), float("inf")), (1, 3, float("inf"), float("nan")),
                          (2, 3, float("nan"), float("nan")), (2, 68, None, float("inf"))):
        pos = lens[i] + node
        page = int(c.table[i, pos // 16])
        if k is not None:
            c.k[page, pos % 16] = k
            c.ks[i][pos] = k
        c.v[page, pos % 16, :, ::3] = v
        c.vs[i][pos, :, ::3] = v
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, mask=pack(masks, 2))
    assert (got[[0, 3, 4]] == 0).all()
    inf_row = got[int(c.start[2]) + 69].double()
    assert torch.isinf(inf_row[:, ::3]).all() and (inf_row[:, ::3] > 0).all()
    keep = [x for x in range(64) if x % 3]
    assert torch.isfinite(inf_row[:, keep]).all()
    got[int(c.start[2]) + 69] = 0
    masks[2][69] = False
    c.ks[0][3] = c.ks[1][203] = c.ks[2][3] = 0    # seen by nobody: the formula's 0 * NaN is not the kernel's
    sees = [np.concatenate([np.ones((t, p), bool), m], 1) for t, p, m in zip(nodes, lens, masks)]
    check(c, got, sees, qt)


@pytest.mark.parametrize("qt,ct", [("bf16", "bf16"), ("f32", "f32"), ("f32", "f16")])
def test_refused_requests_and_bad_pages(cuda, qt, ct):
    """Requests that the plan refused (kv_len 0), with more nodes than the
    mask's words, with more positions than their table, or whose node range
    leaves the token rows, are zero or left; pages outside the pool count as
    masked; rows behind the last request stay as they were."""
    import bml_b200
    lens, nodes = [300, 50, 90, 100, 33], [5, 70, 4, 6, 3]
    c = Paged(lens, nodes, 8, 2, 128, 16, qt, ct, seed=13, spare_rows=4)
    kv = c.kv_lens.clone()
    kv[0] = 0
    kv[2] = c.table.shape[1] * 16 + 1
    c.table[3, 2] = c.k.shape[0]        # positions 32..47
    c.table[3, 4] = -5                  # 64..79
    out = torch.full_like(c.q, 7.0)
    masks = [np.tril(np.ones((t, t), bool)) for t in nodes]
    m = torch.cat([pack(masks, 2)[:, :1], torch.zeros(4, 1, dtype=torch.int64, device="cuda")]).contiguous()
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, kv, c.start, mask=m, out=out)
    s = c.start.tolist()
    assert (got[:s[3]] == 0).all()
    assert (got[s[5]:] == 7).all()
    see = chain(6, 100)
    see[:, 32:48] = see[:, 64:80] = False
    check(c, got, [None, None, None, see, chain(3, 33)], qt, only=[3, 4])
    # a request all of whose pages are bad sees nothing
    c.table[4] = 1 << 30
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, kv, c.start, mask=m, out=out)
    assert (got[s[4]:s[5]] == 0).all()
    # node ranges that leave the rows, or run backwards, write nothing
    bad = c.start.clone()
    bad[5] = 1000
    out.fill_(7.0)
    bml_b200.tree_attention(c.q, c.k, c.v, c.table, kv, bad, mask=m, out=out)
    assert (out[s[4]:] == 7).all()
    check(c, out, [None, None, None, see], qt, only=[3])


def test_offsets_past_32_bits(cuda):
    """Pages at the end of a pool of more than 2^31 elements (4.5 GB)."""
    import bml_b200
    c = Paged([200, 31], [9, 1], 8, 8, 128, 64, "bf16", "bf16", seed=14)
    n_pages = (1 << 31) // (64 * 8 * 128) + 40
    k = torch.empty(n_pages, 64, 8, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    used = c.k.shape[0]
    k[-used:], v[-used:] = c.k, c.v
    table = torch.where(c.table >= 0, c.table + (n_pages - used), c.table).int()
    for q in (c.q, c.q.float()):
        got = bml_b200.tree_attention(q, k, v, table, c.kv_lens, c.start)
        want = bml_b200.tree_attention(q, c.k, c.v, c.table, c.kv_lens, c.start)
        assert torch.equal(got, want)
    check(c, want, [chain(9, 200), chain(1, 31)], "f32")
    q2, k2, v2 = (torch.randn(3, 8, 128, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    last = n_pages * 64 - 1
    bml_b200.paged_append(q2, k2, v2, torch.tensor([last, -1, n_pages * 64], device="cuda"), None, k, v)
    assert torch.equal(k[-1, -1], k2[0]) and torch.equal(v[-1, -1], v2[0])


def test_more_requests_than_one_launch(cuda):
    import bml_b200
    lens = [i % 37 for i in range(1500)]
    c = Paged(lens, [1] * 1500, 4, 2, 64, 16, "bf16", "bf16", seed=15)
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start)
    check(c, got, [chain(1, p) for p in lens], "bf16", only=[0, 1, 700, 1023, 1024, 1025, 1499])


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (128, 128)])
def test_wide_tables(cuda, qt, ct, d, page):
    """Tables far wider than the requests (the kernels for much work): rows that
    see nothing, values that are not finite in nodes that a row does not see and
    in one that it sees, and pages outside the pool."""
    import bml_b200
    lens, nodes = [0, 200, 0, 300, 129], [6, 7, 70, 20, 64]
    c = Paged(lens, nodes, 8, 2, d, page, qt, ct, seed=14)
    c.table = torch.cat([c.table, torch.full((5, 16384 // page), -1, dtype=torch.int32, device="cuda")], 1).contiguous()
    rng = np.random.default_rng(2)
    masks = [np.zeros((6, 6), bool), np.tril(np.ones((7, 7), bool))] + [rng.random((t, t)) < 0.3 for t in nodes[2:]]
    masks[0][1, 0] = masks[0][2, 5] = masks[0][5, 5] = True   # rows 0, 3, 4 see nothing
    masks[1][:, 3] = masks[2][:, 3] = False                    # NaN: by nobody
    masks[2][:, 67:] = False
    masks[2][69, 68] = True                                    # an infinity: by row 69 only
    for i, node, k, v in ((1, 3, float("inf"), float("nan")), (2, 3, float("nan"), float("nan")), (2, 68, None, float("inf"))):
        pos = lens[i] + node
        at = int(c.table[i, pos // page])
        if k is not None:
            c.k[at, pos % page] = k
        c.v[at, pos % page, :, ::3] = v
        c.ks[i][pos] = 0 if k is not None else c.ks[i][pos]    # seen by nobody: the formula's 0 * NaN is not the kernel's
        c.vs[i][pos, :, ::3] = v
    c.table[3, 1] = c.k.shape[0]                               # positions page .. 2 page - 1
    call = lambda: bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, mask=pack(masks, 2))
    got = call()
    assert torch.equal(got.view(torch.uint8), call().view(torch.uint8))
    assert (got[[0, 3, 4]] == 0).all()
    row = int(c.start[2]) + 69
    assert torch.isposinf(got[row, :, ::3]).all()
    assert torch.isfinite(got[row][:, [x for x in range(d) if x % 3]]).all()
    got[row] = 0
    masks[2][69] = False
    sees = [np.concatenate([np.ones((t, p), bool), m], 1) for t, p, m in zip(nodes, lens, masks)]
    sees[3][:, page:2 * page] = False
    check(c, got, sees, qt)


@pytest.mark.parametrize("qt,ct", [("bf16", "bf16"), ("f32", "f16")])
def test_streams_and_graphs(cuda, qt, ct):
    """Another stream; two graphs whose replays overlap on two streams."""
    import bml_b200
    cs = [Paged([3000, 10, 77], [8, 3, 1], 8, 2, 128, 64, qt, ct, seed=s) for s in (20, 21)]
    want = [bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start) for c in cs]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = bml_b200.tree_attention(cs[0].q, cs[0].k, cs[0].v, cs[0].table, cs[0].kv_lens, cs[0].start, stream=s)
    s.synchronize()
    assert torch.equal(got, want[0])
    graphs, outs = [], []
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    # new lengths in the same graph: the sizes live on the device
    c = cs[0]
    c.kv_lens.copy_(ints([2500, 10, 60]))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start))


@pytest.mark.parametrize("d", [64, 128])
def test_wide_f32_on_streams(cuda, d):
    """32-bit pages with many rows: two graphs replayed on two streams at once,
    one behind the other's plan-like writes of its lengths."""
    import bml_b200
    cs = [Paged([2000, 10, 700] * 5, [20, 8, 30] * 5, 8, 2, d, 16, "f32", "f32", seed=s) for s in (22, 23)]
    want = [bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start) for c in cs]
    check(cs[0], want[0], [chain(t, p) for t, p in zip(cs[0].nodes, cs[0].lens)], "f32")
    full = [c.kv_lens.clone() for c in cs]
    graphs, outs = [], []
    for c, f in zip(cs, full):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.kv_lens.zero_()
            bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start)
            c.kv_lens.copy_(f)
            outs.append(bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start))
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


@pytest.mark.parametrize("qt,ct", TYPES)
def test_uneven_batches(cuda, qt, ct):
    """Batches whose average picks a kernel for few rows, with requests of many
    (several row groups a head), and the other way round."""
    import bml_b200
    rng = np.random.default_rng(40)
    for nodes in ([1] * 60 + [100, 9, 33], [8] * 20 + [256, 0, 70], [256, 256, 1, 0, 5, 64, 60]):
        lens = [int(x) for x in rng.integers(0, 700, len(nodes))]
        c = Paged(lens, nodes, 8, 2, 64, 32, qt, ct, seed=len(nodes))
        masks = [mask_of(random_parents(rng, t)) for t in nodes]
        sees = [np.concatenate([np.ones((t, p), bool), m.reshape(t, t)], 1) for t, p, m in zip(nodes, lens, masks)]
        got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, mask=pack(masks, 4))
        check(c, got, sees, qt)


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("heads,kv", [(160, 1), (96, 1), (7, 7), (40, 8), (6, 2), (24, 12)])
def test_head_groups(cuda, qt, ct, heads, kv):
    """Groups of 1 to 160 q heads a kv head, kv heads that no power of two divides."""
    import bml_b200
    for nodes in ([1, 1, 1], [30, 2, 17]):
        lens = [200, 0, 513]
        c = Paged(lens, nodes, heads, kv, 64, 16, qt, ct, seed=heads)
        got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start)
        check(c, got, [chain(t, p) for t, p in zip(nodes, lens)], qt)


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("nodes", [[1, 1], [4, 4], [40, 40]])
def test_scales(cuda, qt, ct, nodes):
    """A scale of 0 (the mean of what a row sees), a tiny and a large one."""
    import bml_b200
    lens = [150, 5]
    c = Paged(lens, nodes, 8, 2, 128, 16, qt, ct, seed=41)
    for scale in (0.0, 1e-20, 0.7):
        got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, scale=scale)
        check(c, got, [chain(t, p) for t, p in zip(nodes, lens)], qt, scale=scale)


@pytest.mark.parametrize("ct", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("nodes", [[1, 1], [4, 4], [40, 40]])
@pytest.mark.parametrize("size,scale", [(0.0, 1e-30), (2.0 ** -100, 2.0 ** 97), (2.0 ** 118, 2.0 ** -121)])
def test_ranges_of_queries(cuda, ct, nodes, size, scale):
    """32-bit queries of any size, and rows of zeros beside a tiny scale."""
    import bml_b200
    lens = [150, 5]
    c = Paged(lens, nodes, 8, 2, 128, 16, "f32", ct, seed=43)
    c.q *= size
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, scale=scale)
    check(c, got, [chain(t, p) for t, p in zip(nodes, lens)], "f32", scale=scale)


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("nodes", [[1, 1, 1], [3, 2, 5], [40, 40, 3]])
def test_nan_that_is_seen(cuda, qt, ct, nodes):
    """A NaN in a committed K row makes its head's rows of that request NaN, one
    in a V row the same dims of them; a NaN query its own row; nothing else."""
    import bml_b200
    lens = [300, 300, 300]
    for where in range(0, 300, 37):
        c = Paged(lens, nodes, 4, 2, 64, 16, qt, ct, seed=42)
        page = int(c.table[0, where // 16])
        c.k[page, where % 16, 1, 5] = float("nan")
        page = int(c.table[1, where // 16])
        c.v[page, where % 16, 0, 7] = float("nan")
        c.q[-1, 2] = float("nan")
        got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start)
        want = torch.zeros_like(got, dtype=torch.bool)
        s = c.start.tolist()
        want[:s[1], 2:] = True            # q heads 2, 3 read kv head 1
        want[s[1]:s[2], :2, 7] = True
        want[-1, 2] = True
        assert torch.equal(torch.isnan(got), want)


def test_two_streams_at_once(cuda):
    """Eager calls of every form on two streams, neither waiting for the other."""
    import bml_b200
    cases = [Paged([900, 30, 77], nodes, 8, 2, 128, 64, qt, ct, seed=s)
             for s, (nodes, qt, ct) in enumerate([([1, 1, 1], "bf16", "bf16"), ([9, 3, 8], "f16", "f16"),
                                                  ([50, 60, 3], "bf16", "bf16"), ([9, 3, 8], "f32", "f32"),
                                                  ([1, 1, 1], "f32", "bf16")])]
    call = lambda c, st=None: bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, stream=st)  # noqa: E731
    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(10):
        for st in streams:
            got.append([call(c, st) for c in cases])
    torch.cuda.synchronize()
    for g in got:
        for x, w in zip(g, want):
            assert torch.equal(x, w)


# ---------------------------------------------------------------------------
# page_plan
# ---------------------------------------------------------------------------
def plan_reference(lens, new, owned, table, free, used, page, n_tokens, parents, words):
    n, mp = len(lens), table.shape[1]
    table = table.copy()
    start, kv, own_out, status = [0], [], [], []
    slots, pos, masks = [-1] * n_tokens, [0] * n_tokens, [[0] * words for _ in range(n_tokens)]
    cum, took, at = 0, 0, 0
    for i in range(n):
        need = -(-(lens[i] + new[i]) // page)
        first = at
        at += max(new[i], 0)
        start.append(min(at, n_tokens))
        st = 0
        if lens[i] < 0 or new[i] < 0 or owned[i] < 0 or owned[i] > mp or need > mp or \
                (parents is not None and new[i] > 64 * words):
            st = 2
        elif at > n_tokens:
            st = 4
        else:
            add = max(0, need - owned[i])
            base = used + cum
            cum += add
            if add and cum > len(free) - used:
                st = 1
            elif add:
                table[i, owned[i]:need] = free[base:base + add]
                took = cum
        status.append(st)
        kv.append(0 if st else lens[i] + new[i])
        own_out.append(owned[i] if st else max(owned[i], need))
        if st == 0:
            bits = []
            for j in range(new[i]):
                p = lens[i] + j
                slots[first + j] = int(table[i, p // page]) * page + p % page
                pos[first + j] = p
                if parents is not None:
                    a = parents[first + j]
                    b = (bits[a] if 0 <= a < j else 0) | 1 << j
                    bits.append(b)
                    pos[first + j] = lens[i] + bin(b).count("1") - 1
                    masks[first + j] = [(b >> 64 * w) & (2 ** 64 - 1) for w in range(words)]
    return table, start, kv, own_out, used + took, slots, pos, status, masks


@pytest.mark.parametrize("seed", range(12))
def test_plan_matches_reference(cuda, seed):
    import bml_b200
    rng = np.random.default_rng(seed)
    tree = seed % 2 == 0
    words = [1, 2, 4][seed % 3]
    page = [16, 32, 1024][seed % 3]
    n = [1, 3, 40, 257, 1000, 4096][seed % 6]
    hi = 64 * words if tree else 300
    lens = rng.integers(0, 500, n)
    new = rng.integers(0, hi + 1, n) * (rng.random(n) < 0.8)
    owned = -(-lens // page) + rng.integers(0, 2, n)
    if n > 30:
        lens[3], new[5], owned[7] = -1, -4, -2
        lens[11] = 100000
        new[17] = 64 * words + 1
    mp = int((2000 + page - 1) // page)
    need = int(np.maximum(0, -(-(lens + new) // page) - owned)[owned >= 0].sum())
    used = int(rng.integers(0, 10))
    free = rng.permutation(max(1, used + (need if seed % 4 else need // 2)))
    table = rng.integers(0, 1000, (n, mp))
    n_tokens = int(np.maximum(new, 0).sum()) + [0, 5, -20][seed % 3]
    n_tokens = max(n_tokens, 0)
    parents = rng.integers(-2, 70, n_tokens) if tree else None
    args = [ints(lens), ints(new), ints(owned), ints(table), ints(free), ints([used])]
    keep = [a.clone() for a in args]
    p = bml_b200.page_plan(*args, page, n_tokens, parents=ints(parents) if tree else None, n_words=words)
    w = plan_reference(lens.tolist(), new.tolist(), owned.tolist(), table, free.tolist(), used, page, n_tokens,
                       parents.tolist() if tree else None, words)
    assert np.array_equal(args[3].cpu().numpy(), w[0])
    for got, want in ((p.node_start, w[1]), (p.kv_lens, w[2]), (p.owned, w[3]), (p.free_used, [w[4]]),
                      (p.slots, w[5]), (p.positions, w[6]), (p.status, w[7])):
        assert got.tolist() == want
    if tree and n_tokens:
        assert np.array_equal(p.mask.cpu().numpy().view(np.uint64), np.array(w[8], np.uint64))
    for a, b in zip(args[:3] + args[4:], keep[:3] + keep[4:]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n,page", [(1, 16), (3, 64), (40, 16), (300, 128), (300, 16)])
def test_plan_of_prompts(cuda, n, page):
    """Long runs of tokens without drafts: runs that end inside a page or a
    request, requests of none to three tokens between long ones."""
    import bml_b200
    rng = np.random.default_rng(n + page)
    lens = rng.integers(0, 300, n)
    new = np.where(rng.random(n) < 0.5, rng.integers(0, 4, n), rng.integers(0, 700, n))
    own = -(-lens // page) + rng.choice([0, 0, 1, 5], n)
    need = -(-(lens + new) // page)
    width = int(max(own.max(), need.max())) + 1
    pages = rng.permutation(int(own.sum() + np.maximum(need - own, 0).sum()) + 5)
    table, at = np.full((n, width), -1, np.int64), 0
    for i in range(n):
        table[i, :own[i]] = pages[at:at + own[i]]
        at += own[i]
    table = ints(table)
    total = int(new.sum()) + int(rng.integers(0, 9))
    plan = bml_b200.page_plan(ints(lens), ints(new), ints(own), table, ints(pages), ints([at]), page, total)
    plan.check()
    pos = np.concatenate([np.arange(l, l + w) for l, w in zip(lens, new)])
    who = np.repeat(np.arange(n), new)
    slots = table.cpu().numpy().astype(np.int64)[who, pos // page] * page + pos % page
    assert (slots >= 0).all() and len(set(slots.tolist())) == len(slots)
    pad = total - len(pos)
    assert plan.slots.tolist() == slots.tolist() + [-1] * pad
    assert plan.positions.tolist() == pos.tolist() + [0] * pad


# ---------------------------------------------------------------------------
# paged_append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16"),
                                     ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("n,heads,kv,d", [(1, 32, 4, 64), (37, 8, 8, 128), (700, 5, 1, 128), (9, 3, 1, 6), (65, 2, 2, 250)])
def test_append_matches_f64(cuda, src, dst, n, heads, kv, d):
    """Rotation within 2^-24 of sine and cosine (each product off by that much
    of its size) plus one rounding of the sum and one to the destination."""
    import bml_b200
    g = torch.Generator(device="cuda").manual_seed(n + d)
    rng = np.random.default_rng(n)
    page = 16
    n_pages = -(-n // page) + 3
    q, k, v = (torch.randn(n, h, d, device="cuda", generator=g).to(DT[src]) for h in (heads, kv, kv))
    kp, vp = (torch.randn(n_pages, page, kv, d, device="cuda", generator=g).to(DT[dst]) for _ in range(2))
    slots = torch.from_numpy(rng.permutation(n_pages * page)[:n]).cuda()
    pos = torch.from_numpy(rng.integers(0, 200000, n).astype(np.int32)).cuda()
    if n > 5:
        slots[2], slots[4] = -1, n_pages * page
    live = (slots >= 0) & (slots < n_pages * page)
    ang = pos.double()[:, None] * 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]

    def turned(x):
        a, b = x.double()[..., 0::2], x.double()[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        size = torch.stack((a.abs() + b.abs(),) * 2, -1).flatten(-2)
        return y, size

    def close(got, want, size, t):
        lim = 3 * 2.0 ** -24 * size + torch.finfo(DT[t]).eps / 2 * want.abs() + torch.finfo(DT[t]).tiny
        assert ((got.double() - want).abs() <= lim).all()

    q0, kp0, vp0 = q.clone(), kp.clone(), vp.clone()
    q_out = torch.full_like(q, 3.0)
    got = bml_b200.paged_append(q, k, v, slots, pos, kp, vp, q_out=q_out)
    assert got is q_out and torch.equal(q, q0)
    wq, sq = turned(q)
    close(q_out[live], wq[live], sq[live], src)
    assert (q_out[~live] == 3).all()
    wk, sk = turned(k)
    s = slots[live]
    close(kp.view(-1, kv, d)[s], wk[live], sk[live], dst)
    assert torch.equal(vp.view(-1, kv, d)[s], v[live].to(DT[dst]))
    rest = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
    rest[s] = False
    assert torch.equal(kp.view(-1, kv, d)[rest], kp0.view(-1, kv, d)[rest])
    assert torch.equal(vp.view(-1, kv, d)[rest], vp0.view(-1, kv, d)[rest])
    # in place, and without rotation or queries
    q1 = q.clone()
    assert bml_b200.paged_append(q1, k, v, slots, pos, kp, vp) is q1
    assert torch.equal(q1[live], q_out[live]) and torch.equal(q1[~live], q[~live])
    assert bml_b200.paged_append(None, k, v, slots, None, kp, vp) is None
    assert torch.equal(kp.view(-1, kv, d)[s], k[live].to(DT[dst]))


# ---------------------------------------------------------------------------
# paged_commit
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt,kv,d,page", [("bf16", 8, 128, 64), ("f16", 4, 64, 16), ("f32", 3, 6, 32), ("bf16", 1, 3, 16)])
def test_commit_matches_moves(cuda, dt, kv, d, page):
    import bml_b200
    rng = np.random.default_rng(d)
    lens, nodes = [0, 5, 16, 100, 30, 7, 12], [4, 20, 64, 200, 0, 9, 6]
    paths = [[0, 1, 3], [2, 5, 6, 19], [0, 1, 2], sorted(rng.permutation(200)[:40].tolist()), [0], [3, 3, 5], [4, 6]]
    kept = [3, 4, 3, 40, 0, 1, 1]                # a path ends where it stops growing, or leaves the nodes
    total = [a + b for a, b in zip(lens, nodes)]
    need = [-(-t // page) for t in total]
    order = rng.permutation(sum(need) + 1)
    table = np.zeros((7, max(need)), np.int64)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c]
        at += c
    kp = torch.randn(3, sum(need) + 1, page, kv, d, device="cuda").to(DT[dt])
    vp = torch.randn_like(kp)
    want = [kp.clone(), vp.clone()]
    for w in want:
        rows = w.view(3, -1, kv, d)
        for i in range(7):
            for j in range(kept[i]):
                a, b = lens[i] + paths[i][j], lens[i] + j
                rows[:, table[i, b // page] * page + b % page] = rows[:, table[i, a // page] * page + a % page].clone()
    wide = max(len(x) for x in paths)
    path = ints([x + [0] * (wide - len(x)) for x in paths])
    ln, kv_lens = ints(lens), ints(total)
    got = bml_b200.paged_commit(kp, vp, ints(table), ln, kv_lens, starts_of(nodes), path, ints([len(x) for x in paths]))
    assert got.tolist() == [a + b for a, b in zip(lens, kept)]
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    # refused requests keep their lengths and rows
    got = bml_b200.paged_commit(kp, vp, ints(table), ln, torch.zeros_like(kv_lens), starts_of(nodes), path,
                                ints([len(x) for x in paths]))
    refused = [a for a, b in zip(lens, nodes)]
    assert got.tolist() == refused
    assert torch.equal(kp, want[0])


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("qt,ct", [("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
def test_batcher_run(cuda, qt, ct):
    """Requests join with prompts, draft trees, keep a path, decode single
    tokens and leave; each step's attention against the formula over a cache
    kept per request, rows in the cache against the appended ones."""
    import bml_b200
    rng = np.random.default_rng(4)
    layers, heads, kv, d = 2, 8, 2, 64
    b = bml_b200.PagedBatcher(layers, heads, kv, d, n_pages=40, page_size=16, max_positions=256, dtype=DT[ct],
                              max_requests=4)
    kept = {}

    def admit(rid, prompt):
        k, v = (torch.randn(layers, prompt, kv, d, device="cuda").to(DT[ct]) for _ in range(2))
        b.add(rid, k if prompt else None, v if prompt else None)
        kept[rid] = (k, v)

    admit("a", 0)
    admit("b", 33)
    admit("c", 100)
    for step in range(8):
        if step == 3:
            b.remove("b")
            del kept["b"]
            admit("d", 48)
            admit("e", 15)
        if step == 6:
            b.remove("c")
            del kept["c"]
        new = {}
        for rid in b.active:
            t = int(rng.integers(1, 20))
            new[rid] = random_parents(rng, t) if step % 2 else (t if step == 4 else 1)
        if step == 5:
            del new["a"]
        plan = b.begin(new)
        rows = [r for r in b.active if r in new]
        trees = {r: (list(range(-1, x - 1)) if isinstance(x, int) else x) for r, x in new.items()}
        n = sum(len(trees[r]) for r in rows)
        drafted = {r: ([], []) for r in rows}
        for layer in range(layers):
            q = torch.randn(n, heads, d, device="cuda").to(DT[qt])
            k, v = (torch.randn(n, kv, d, device="cuda").to(DT[qt]) for _ in range(2))
            out = b.step(layer, q, k, v)
            at = 0
            for r in rows:
                t, p = len(trees[r]), kept[r][0].shape[1]
                m = mask_of(trees[r])
                depth = m.sum(1) - 1
                assert plan.positions[at:at + t].tolist() == [p + int(x) for x in depth]
                ang = torch.tensor(p + depth, device="cuda").double()[:, None] * 10000.0 ** (
                    -torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
                x = k[at:at + t].double()
                c, s = ang.cos()[:, None], ang.sin()[:, None]
                kt = torch.stack((x[..., 0::2] * c - x[..., 1::2] * s, x[..., 0::2] * s + x[..., 1::2] * c), -1)
                drafted[r][0].append(kt.flatten(-2).to(DT[ct]))
                drafted[r][1].append(v[at:at + t].to(DT[ct]))
                case = object.__new__(Paged)
                case.ks = [torch.cat([kept[r][0][layer], drafted[r][0][layer]])]
                case.vs = [torch.cat([kept[r][1][layer], drafted[r][1][layer]])]
                case.q, case.start, case.nodes, case.lens, case.group = q[at:at + t], [0], [t], [p], heads // kv
                sees = np.concatenate([np.ones((t, p), bool), m], 1)
                want, ab, bm = case.want(0, sees)
                # a 16-bit K row may be rounded the other way where the f64 and f32 rotations straddle a step
                slack = 0 if ct == "f32" else bm * torch.finfo(DT[ct]).eps * ab
                lim = tol(qt, want, ab, bm) + slack + (1e-5 * ab if ct == "f32" else 0)
                assert ((out[at:at + t].double() - want).abs() <= lim).all()
                at += t
        paths = {}
        for r in rows:
            t = len(trees[r])
            m = mask_of(trees[r])
            if step % 2:
                paths[r] = [int(a) for a in np.flatnonzero(m[int(rng.integers(0, t))])]
            keep = paths.get(r, list(range(t)))
            kept[r] = tuple(torch.cat([kept[r][i], torch.stack(drafted[r][i])[:, keep]], 1) for i in range(2))
        b.commit(paths)
        for r in b.active:
            assert b.length(r) == kept[r][0].shape[1]
            for layer in range(layers):
                kc, vc = b.cache(r, layer)
                eps = torch.finfo(DT[ct]).eps
                assert ((kc.double() - kept[r][0][layer].double()).abs() <= eps * 2 * kc.double().abs() + 1e-5).all()
                assert torch.equal(vc, kept[r][1][layer])
    # every page is held once or free
    used = int(b.used)
    held = [p for r in b.active for p in b.table[b._rows[r], :int(b.owned[b._rows[r]])].tolist()]
    assert sorted(held) == sorted(b.free[:used].tolist())
    assert sorted(held + b.free[used:].tolist()) == list(range(40))


def test_empty_steps(cuda):
    """No request at all, requests without new tokens, and a request without a
    prompt whose first step is a draft."""
    import bml_b200
    b = bml_b200.PagedBatcher(1, 4, 2, 64, n_pages=8, page_size=16, max_positions=64, max_requests=3)
    none = [torch.empty(0, h, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2, 2)]
    for _ in range(2):
        plan = b.begin({})
        assert plan.slots.numel() == 0 and plan.node_start.tolist() == [0] * 4
        assert b.step(0, *none).shape == (0, 4, 64)
        b.commit()
        if not len(b):
            b.add("x")
            b.add("y")
    plan = b.begin({"y": [-1, -1, 0, 2]})
    assert plan.node_start.tolist() == [0, 0, 4, 4] and plan.positions.tolist() == [0, 0, 1, 2]
    q, k, v = (torch.randn(4, h, 64, device="cuda").bfloat16() for h in (4, 2, 2))
    out = b.step(0, q, k, v)
    want = v[:2].repeat_interleave(2, 1)      # a root sees itself only
    assert torch.equal(out[:2], want)
    b.commit({"y": []})
    assert b.length("x") == b.length("y") == 0
    b.remove("y")
    b.remove("x")
    assert len(b) == 0 and int(b.used) == 0 and sorted(b.free.tolist()) == list(range(8))


def test_batcher_limits(cuda):
    import bml_b200
    b = bml_b200.PagedBatcher(1, 4, 2, 64, n_pages=3, page_size=16, max_positions=64, max_requests=2)
    b.add(0)
    b.add(1)
    with pytest.raises(bml_b200.AtCapacity):
        b.add(2)
    with pytest.raises(KeyError):
        b.add(1)
    with pytest.raises(bml_b200.OutOfPages):
        b.begin({0: 33, 1: 1})
    with pytest.raises(bml_b200.OutOfPages):
        b.begin({0: 65})
    with pytest.raises(ValueError):
        b.begin({0: 257})
    with pytest.raises(RuntimeError):
        b.commit()
    b.begin({0: 20, 1: [-1, 0, 0]})
    with pytest.raises(RuntimeError):
        b.begin({0: 1})
    q = torch.zeros(23, 4, 64, device="cuda", dtype=torch.bfloat16)
    kv = torch.zeros(23, 2, 64, device="cuda", dtype=torch.bfloat16)
    b.step(0, q, kv, kv)
    with pytest.raises(ValueError):
        b.commit({1: [1, 1]})
    with pytest.raises(ValueError):
        b.commit({1: [3]})
    b.commit({1: [0, 2]})
    assert b.length(0) == 20 and b.length(1) == 2
    b.remove(0)
    b.begin({1: 40})
    b.commit()
    assert b.length(1) == 42


def test_batcher_prompt_that_fails(cuda):
    """A prompt that cannot be stored leaves no request and takes no pages."""
    import bml_b200
    b = bml_b200.PagedBatcher(1, 4, 2, 64, n_pages=3, page_size=16, max_positions=64, max_requests=2)
    x = torch.zeros(1, 20, 2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        b.add("a", x.double(), x.double())
    with pytest.raises(ValueError):
        b.add("a", x.cpu(), x.cpu())
    with pytest.raises(bml_b200.OutOfPages):
        b.add("a", x.repeat(1, 3, 1, 1), x.repeat(1, 3, 1, 1))
    assert len(b) == 0 and int(b.used) == 0
    b.add("a", x, x)
    assert b.length("a") == 20 and int(b.used) == 2


# ---------------------------------------------------------------------------
# The two ways of the Python wrappers
# ---------------------------------------------------------------------------
class _Leaves:
    """Stands for the binding in C++ and leaves every call to the wrappers."""

    def __getattr__(self, name):
        return lambda *a: None


def _all_calls():
    import bml_b200
    c = Paged([40, 3], [3, 1], 4, 2, 64, 16, "bf16", "bf16", seed=30)
    free, used = ints(list(range(20))), ints([0])
    p = bml_b200.page_plan(ints([0, 5]), ints([3, 20]), ints([0, 1]), c.table.clone(), free, used, 16, 25,
                           parents=ints([-1, 0, 0] + list(range(-1, 19)) + [0, 0]), n_words=2)
    outs = [p.node_start, p.kv_lens, p.owned, p.free_used, p.status, p.positions, p.slots, p.mask]
    p = bml_b200.page_plan(ints([0, 5]), ints([3, 20]), ints([0, 1]), c.table.clone(), free, used, 16, 23)
    outs += [p.positions, p.slots]
    assert p.mask is None
    kp, vp = torch.zeros(3, 16, 2, 64, device="cuda"), torch.zeros(3, 16, 2, 64, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(31)
    q, k, v = (torch.randn(4, h, 64, device="cuda", generator=g) for h in (4, 2, 2))
    slots, pos = torch.tensor([1, -1, 40, 7], device="cuda"), ints([5, 6, 7, 100000])
    q2 = torch.empty_like(q).fill_(1)
    assert bml_b200.paged_append(q, k, v, slots, pos, kp, vp, q_out=q2) is q2
    assert bml_b200.paged_append(None, k, v, slots, None, vp, kp) is None
    outs += [q2, kp, vp]
    outs.append(bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start))
    outs.append(bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, scale=0.3, mask=torch.full(
        (4, 1), 5, dtype=torch.int64, device="cuda")))
    kc, vc = c.k[None].nan_to_num().contiguous(), c.v[None].nan_to_num().contiguous()
    outs.append(bml_b200.paged_commit(kc, vc, c.table, ints([40, 3]), c.kv_lens, c.start, ints([[0, 2], [0, 0]]), ints([2, 1])))
    return outs + [kc, vc]


def test_both_ways_agree(cuda, monkeypatch):
    """The binding in C++ and the wrappers' own way give the same bits."""
    import bml_b200.paged as P
    a = _all_calls()
    assert P._fast is not None
    monkeypatch.setattr(P, "_fast", _Leaves())
    b = _all_calls()
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)


def test_refusals_of_gpu_tensors(cuda):
    """What either way must not let through: another type, shape, device or
    layout, and what the C call refuses."""
    import bml_b200
    c = Paged([40, 3], [3, 1], 4, 2, 64, 16, "bf16", "bf16", seed=32)
    t = bml_b200.tree_attention
    good = (c.q, c.k, c.v, c.table, c.kv_lens, c.start)
    assert t(*good).shape == c.q.shape

    def bad(i, x, err=ValueError, **kw):
        args = list(good)
        if i is not None:
            args[i] = x
        with pytest.raises(err):
            t(*args, **kw)

    bad(0, c.q.double(), TypeError)
    bad(0, c.q.half(), bml_b200.BmlUnsupported)
    bad(0, c.q.transpose(0, 1).contiguous().transpose(0, 1))
    bad(0, c.q[:, :3].contiguous(), bml_b200.BmlInvalid)          # 3 heads over 2
    bad(0, torch.cat([c.q, c.q], 2), ValueError)
    bad(0, c.q.cpu())
    bad(1, c.k.float(), TypeError)
    bad(1, c.k[:, :8].contiguous())
    bad(2, c.v[:1])
    bad(3, c.table.long(), TypeError)
    bad(3, c.table[:1])
    bad(4, c.kv_lens[:1])
    bad(4, c.kv_lens.long(), TypeError)
    bad(5, c.start[:2])
    bad(None, None, mask=torch.zeros(4, 1, dtype=torch.int32, device="cuda"), err=TypeError)
    bad(None, None, mask=torch.zeros(3, 1, dtype=torch.int64, device="cuda"))
    bad(None, None, mask=torch.zeros(4, 5, dtype=torch.int64, device="cuda"))
    bad(None, None, scale=float("nan"), err=bml_b200.BmlInvalid)
    bad(None, None, out=c.q, err=bml_b200.BmlInvalid)
    bad(None, None, out=torch.empty_like(c.q[:2]))
    bad(None, None, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"), err=bml_b200.BmlInvalid)
    odd = torch.empty(c.k.numel() + 1, dtype=c.k.dtype, device="cuda")[1:].view(c.k.shape)
    bad(1, odd, bml_b200.BmlInvalid)                               # pool off a 16-byte boundary
    wide = torch.zeros(4, 4, 96, device="cuda", dtype=torch.bfloat16)
    pool = torch.zeros(4, 16, 2, 96, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(bml_b200.BmlUnsupported):
        t(wide, pool, pool, *good[3:])
    i2 = ints([1, 1])
    with pytest.raises(ValueError):
        bml_b200.page_plan(i2, ints([1]), i2, c.table, i2, ints([0]), 16, 2)
    with pytest.raises(bml_b200.BmlInvalid):
        bml_b200.page_plan(i2, i2, i2, c.table, i2, ints([0]), 17, 2)
    with pytest.raises(ValueError):
        bml_b200.page_plan(i2, i2, i2, c.table, i2, ints([0]), 16, 2, parents=i2, n_words=5)
    with pytest.raises(ValueError):
        bml_b200.page_plan(i2, i2, i2, c.table, i2, ints([0]), 16, -1)
    q, kv = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")
    sl = torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError):
        bml_b200.paged_append(q.half(), kv, kv, sl, i2, c.k, c.v)
    with pytest.raises(ValueError):
        bml_b200.paged_append(q, kv, kv, sl[:1], i2, c.k, c.v)
    with pytest.raises(ValueError):
        bml_b200.paged_append(None, kv, kv, sl, i2, c.k, c.v, q_out=q)
    with pytest.raises(bml_b200.BmlInvalid):
        bml_b200.paged_append(q, kv, kv, sl, i2, c.k, c.v, theta=-1.0)
    with pytest.raises(ValueError):
        bml_b200.paged_commit(c.k[None], c.v[None], c.table, i2, c.kv_lens, c.start, i2, i2)
