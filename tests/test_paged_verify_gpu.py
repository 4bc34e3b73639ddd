"""GPU tests of verify_drafts against a plain Python walk in 64 bits over
include/bml_attn.h's formulas, and of the distribution that the tokens have.

Results are whole numbers.  The walk's sums differ from the kernel's by their
order, at most 2^-52 times the number of terms relatively (1e-10 for the largest
vocabulary here); a decision whose two sides are nearer than that would be left
out, and none is: the tests assert that too."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


class Near(Exception):
    pass


def below(a, b):
    if a != b and abs(a - b) <= 1e-10 * max(abs(a), abs(b)):
        raise Near
    return a < b


def clean(x):
    x = np.asarray(x, np.float64).copy()
    x[~((x > 0) & np.isfinite(x))] = 0
    return x


def walk(p, q, tokens, parents, u, u_next, max_path):
    """path, next token of one request."""
    vocab, t_all = p.shape[1], len(tokens)
    if t_all == 0 or t_all > 256:
        return [], -1
    path, t = [0], 0
    while True:
        pt, c, mass = clean(p[t]), 0.0, 1.0
        qt = None if q is None else clean(q[t])
        kids = [j for j in range(1, t_all) if parents[j] == t and 0 <= parents[j] < j and 0 <= tokens[j] < vocab]
        if len(path) == max_path:
            kids = []
        found = None
        for k, j in enumerate(kids):
            x = tokens[j]
            if q is None:
                if below(float(u[j]) * mass, pt[x]):
                    found = j
                    break
                mass -= pt[x]
                pt[x] = 0.0
            else:
                r = max(pt[x] - c * qt[x], 0.0)
                if below(float(u[j]) * qt[x] * mass, r):
                    found = j
                    break
                c += mass
                if k + 1 < len(kids):
                    mass = math.fsum(np.maximum(pt - c * qt, 0.0))
        if found is None:
            break
        path.append(found)
        t = found
    w = pt if q is None else np.maximum(pt - c * qt, 0.0)
    if w.sum() <= 0:
        if q is not None and qt.sum() > 2 * pt.sum():
            return path, vocab - 1
        w = clean(p[t])
    if w.sum() <= 0:
        return path, vocab - 1
    cum = np.cumsum(w.astype(np.longdouble))
    tau = np.longdouble(float(u_next)) * cum[-1]
    hit = np.flatnonzero(cum > tau)
    nxt = int(hit[0]) if len(hit) else int(np.flatnonzero(w > 0)[-1])
    for edge in (cum[nxt], cum[nxt - 1] if nxt else np.longdouble(0)):
        if edge != tau and abs(edge - tau) < 1e-10 * cum[-1]:
            raise Near
    return path, nxt


def tree(rng, t):
    return [-1] + [int(rng.integers(max(0, j - 4), j)) for j in range(1, t)]


def batch(nodes, vocab, dt, draft, seed, sharp=3.0):
    """Random drafts whose tokens come from the draft rows."""
    rng = np.random.default_rng(seed)
    n = sum(nodes)
    logits = rng.standard_normal((n, vocab)) * sharp
    soft = lambda x: np.exp(x - x.max(1, keepdims=True)) / np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)  # noqa: E731
    p = torch.from_numpy(soft(logits)).to(DT[dt])
    q = torch.from_numpy(soft(logits + rng.standard_normal((n, vocab)))).to(DT[dt])
    parents, tokens, at = [], [], 0
    for t in nodes:
        par = tree(rng, t) if t else []
        parents += par
        for j in range(t):
            row = q[at + max(par[j], 0)].double().numpy()
            if draft:
                tokens.append(int(rng.choice(vocab, p=row / row.sum())))
            else:
                tokens.append(int(np.argsort(-row)[rng.integers(0, min(vocab, 4))]))
        at += t
    u, un = (torch.from_numpy(rng.random(k).astype(np.float32)) for k in (n, len(nodes)))
    return dict(p=p, q=q if draft else None, tokens=tokens, parents=parents, u=u, un=un, nodes=list(nodes))


def call(b, max_path=256, **kw):
    import bml_b200
    start = np.concatenate([[0], np.cumsum(b["nodes"])])
    cu = lambda x: None if x is None else x.cuda()  # noqa: E731
    return bml_b200.verify_drafts(cu(b["p"]), cu(b["q"]), ints(b["tokens"]), ints(b["parents"]), ints(start), cu(b["u"]), cu(b["un"]),
                                  max_path=max_path, **kw)


def check(b, max_path=256, **kw):
    path, count, token = (x.tolist() for x in call(b, max_path, **kw))
    at, near = 0, 0
    for i, t in enumerate(b["nodes"]):
        s = slice(at, at + t)
        try:
            want, nxt = walk(b["p"][s].double().numpy(), None if b["q"] is None else b["q"][s].double().numpy(), b["tokens"][s],
                             b["parents"][s], b["u"][s].numpy(), b["un"][i], max_path)
        except Near:
            near += 1
            at += t
            continue
        assert count[i] == len(want), (i, path[i][:12], want)
        assert path[i] == want + [-1] * (max_path - len(want)), i
        assert token[i] == nxt, (i, want)
        at += t
    assert near == 0
    return path, count, token


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("vocab,nodes", [(1, [1, 3]), (7, [5, 0, 1, 30]), (300, [64, 2, 17]), (1001, [1] * 9), (4096, [12] * 40),
                                         (32001, [9]), (50000, [1, 20, 6])])
def test_walks(cuda, dt, draft, vocab, nodes):
    for seed in range(3 if vocab < 30000 else 1):
        check(batch(nodes, vocab, dt, draft, 10 * seed + vocab), max_path=max(nodes))


@pytest.mark.parametrize("n", [1, 30, 70, 140, 300])
def test_batches_of_every_cluster_size(cuda, n):
    """1, 2, 4 or 8 CTAs a request; the longest drafts and the most siblings."""
    rng = np.random.default_rng(n)
    check(batch([int(x) for x in rng.integers(0, 12, n)], 5003, "f32", n % 2 == 0, n), max_path=12)


@pytest.mark.parametrize("draft", [True, False])
def test_many_nodes(cuda, draft):
    b = batch([256, 257, 3], 600, "f32", draft, 5)
    b["parents"][1:120] = [0] * 119                     # siblings by the score, tokens among them twice
    b["u"][1:110] = 0.999
    path, count, token = check(b)
    assert count[1] == 0 and token[1] == -1
    chain = batch([256], 40, "f32", draft, 6)
    chain["parents"] = list(range(-1, 255))
    chain["u"][:] = 0.0                                 # everything is kept
    assert check(chain)[1] == [256]
    for most in (1, 2, 100):
        assert check(chain, max_path=most)[1] == [most]


@pytest.mark.parametrize("draft", [True, False])
def test_odd_inputs(cuda, draft):
    """Tokens and parents that are none, probabilities that are none, the edges of
    the random numbers, and rows without weight."""
    b = batch([12, 9, 1, 4, 4, 4], 50, "f32", draft, 7, sharp=1.0)
    b["tokens"][3], b["tokens"][4] = -1, 50
    b["parents"][5], b["parents"][6] = 6, 99
    b["parents"][0], b["parents"][12] = 5, -7            # of node 0: not looked at
    b["p"][0, :5] = torch.tensor([float("nan"), float("inf"), -1.0, float("-inf"), 0.0])
    if draft:
        b["q"][0, 2:7] = torch.tensor([float("nan"), float("inf"), -1.0, float("-inf"), 0.0])
    b["un"][0], b["un"][1] = 0.0, 1 - 2.0 ** -24
    b["u"][12:21] = 1 - 2.0 ** -24
    b["p"][22] = 0.0                                     # the fourth request's node 0: nothing to draw
    b["u"][23:26] = 0.5
    b["p"][26], b["p"][30] = 0.0, 0.0
    b["p"][26, 9] = b["p"][30, 9] = 1.0                  # only one token, whose draft is rejected with u = 1
    b["tokens"][27], b["parents"][27], b["u"][27] = 9, 0, 1.0
    b["tokens"][31], b["parents"][31], b["u"][31] = 9, 0, 0.5
    if draft:
        b["q"][26] = b["p"][26]
        b["q"][30] = b["p"][30]
    path, count, token = check(b)
    assert count[3] == 1 and token[3] == 49
    assert count[4] == 1 and token[4] == 9               # nothing is left of the residual: p itself
    assert count[5] >= 2


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_nothing_left_of_a_residual(cuda, dt):
    """Rows whose rounding leaves p below q everywhere: the token comes from p; rows
    that are no distributions (prefix sums here) end at vocab - 1."""
    b = batch([3, 3, 2, 4], 500, dt, True, 12)
    for r, top in ((0, 1.0), (3, 1.0), (6, 0.9)):
        b["p"][r] = 0
        b["q"][r] = 0
        b["q"][r, 77] = top
        b["p"][r, 77] = top * (1 - 2.0 ** -7)
    b["p"][3, 400] = b["q"][3, 400] = 2.0 ** -12
    for j in (1, 2, 4, 5, 7):
        b["tokens"][j], b["u"][j] = 77, 1 - 2.0 ** -20
    b["parents"][:8] = [-1, 0, 0, -1, 0, 0, -1, 0]
    b["q"][8:] = b["p"][8:].float().cumsum(-1).to(DT[dt]) + 0.5
    b["u"][9:] = 0.99
    path, count, token = check(b)
    assert count == [1, 1, 1, 1] and token == [77, 77, 77, 499]
    b["q"] = None
    assert check(b)[2][0] == 77


def test_unaligned_rows(cuda):
    """Rows that start anywhere, and target and draft on different boundaries."""
    import bml_b200
    for dt in DT:
        b = batch([5, 8], 1003, dt, True, 8)
        want = [x.tolist() for x in call(b)]
        start = ints([0, 5, 13])
        for a, c in ((1, 1), (3, 0), (0, 5)):
            p, q = (torch.empty(13 * 1003 + 8, dtype=DT[dt], device="cuda")[k:k + 13 * 1003].view(13, 1003) for k in (a, c))
            p.copy_(b["p"])
            q.copy_(b["q"])
            got = bml_b200.verify_drafts(p, q, ints(b["tokens"]), ints(b["parents"]), start, b["u"].cuda(), b["un"].cuda())
            assert [x.tolist() for x in got] == want


def test_unaligned_rows_with_nothing_left(cuda):
    """q is summed where it lies: draft rows on another boundary than the target's, a
    residual that is empty, and values that are looked at one by one."""
    import bml_b200
    for dt in DT:
        for bump in (0.0, 0.5, float("nan"), float("inf"), -1.0, 7.0):
            b = batch([4, 5], 1003, dt, True, 13)
            b["q"][:4] = b["p"][:4].float() + bump if bump == bump and bump >= 0 and bump != float("inf") else b["p"][:4].float()
            if bump != bump or bump in (float("inf"), -1.0):
                b["q"][:, 5::7] = bump
                b["p"][:, 6::9] = bump
            b["u"][:] = 1.0
            want = check(b)
            for a, c in ((1, 0), (0, 3), (2, 5), (4, 4)):
                p, q = (torch.empty(9 * 1003 + 8, dtype=DT[dt], device="cuda")[k:k + 9 * 1003].view(9, 1003) for k in (a, c))
                p.copy_(b["p"])
                q.copy_(b["q"])
                got = bml_b200.verify_drafts(p, q, ints(b["tokens"]), ints(b["parents"]), ints([0, 4, 9]), b["u"].cuda(), b["un"].cuda())
                assert tuple(x.tolist() for x in got) == tuple(want)


def test_first_token_is_distributed_as_the_target(cuda):
    """The first token behind the pending one -- a kept draft or the drawn one --
    over 200,000 requests with the same rows: each count is binomial, so within
    6 standard deviations of its mean (a chance of 1e-8 for 40 of them)."""
    import bml_b200
    n, vocab = 200_000, 8
    for draft, kids in ((True, 3), (True, 1), (False, 3)):
        g = torch.Generator(device="cuda").manual_seed(kids + draft)
        p0 = torch.tensor([.3, .02, .18, .0, .25, .05, .1, .1], device="cuda")
        q0 = torch.tensor([.1, .3, .1, .1, .2, .0, .15, .05], device="cuda")
        t = kids + 1
        p = p0.repeat(n * t, 1)
        q = q0.repeat(n * t, 1) if draft else None
        tok = torch.zeros(n, t, dtype=torch.int32, device="cuda")
        tok[:, 1:] = (torch.multinomial(q0, n * kids, True, generator=g).view(n, kids) if draft else torch.tensor([4, 0, 1], device="cuda"))
        par = torch.zeros(n, t, dtype=torch.int32, device="cuda")
        par[:, 0] = -1
        start = torch.arange(0, n * t + 1, t, dtype=torch.int32, device="cuda")
        u, un = torch.rand(n * t, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)
        path, count, nxt = bml_b200.verify_drafts(p, q, tok.flatten(), par.flatten(), start, u, un, max_path=2)
        # a path of two nodes ends there; its second is the first token, else the drawn one
        first = torch.where(count == 2, tok.gather(1, path[:, 1:].clamp(min=0).long())[:, 0], nxt)
        got = torch.bincount(first, minlength=vocab).double()
        mean = n * p0.double() / p0.double().sum()
        sd = (mean * (1 - p0.double())).sqrt()
        assert ((got - mean).abs() <= 6 * sd + 1).all(), (draft, kids, got, mean)
        # and the token behind a kept draft is the target's too
        after = nxt[count == 2]
        m2 = len(after) * p0.double()
        assert ((torch.bincount(after, minlength=vocab).double() - m2).abs() <= 6 * m2.sqrt() + 1).all()


def test_streams_graphs_and_both_ways(cuda, monkeypatch):
    import bml_b200
    import bml_b200.paged as P
    b = batch([9, 0, 33, 1], 3001, "bf16", True, 9)
    want = [x.clone() for x in call(b, 40)]
    assert P._fast not in (None, P._Wrappers)
    st = torch.cuda.Stream()
    args = [b["p"].cuda(), b["q"].cuda(), ints(b["tokens"]), ints(b["parents"]), ints([0, 9, 9, 42, 43]), b["u"].cuda(), b["un"].cuda()]
    torch.cuda.synchronize()
    got = bml_b200.verify_drafts(*args, max_path=40, stream=st)
    st.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = bml_b200.verify_drafts(*args, max_path=40)
    u = args[5].clone()
    other = [x.clone() for x in call({**b, "u": torch.ones_like(b["u"])}, 40)]
    for k in range(3):
        args[5].copy_(torch.ones_like(u) if k == 1 else u)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, other if k == 1 else want))
    del g
    monkeypatch.setattr(P, "_fast", P._Wrappers)
    assert all(torch.equal(x, y) for x, y in zip(bml_b200.verify_drafts(*args, max_path=40), want))


def test_refusals_of_gpu_tensors(cuda):
    import bml_b200
    b = batch([3, 2], 40, "f32", True, 1)
    good = [b["p"].cuda(), b["q"].cuda(), ints(b["tokens"]), ints(b["parents"]), ints([0, 3, 5]), b["u"].cuda(), b["un"].cuda()]
    for i, x, err in ((0, good[0].double(), TypeError), (0, good[0].cpu(), ValueError), (0, good[0][None], ValueError),
                      (0, good[0].T.contiguous().T, ValueError), (1, good[1].half(), TypeError), (1, good[1][:4], ValueError),
                      (2, good[2].long(), TypeError), (2, good[2][:4], ValueError), (3, good[3][:1], ValueError),
                      (4, good[4].long(), TypeError), (5, good[5].double(), TypeError), (5, good[5][:2], ValueError),
                      (6, good[6][:1], ValueError), (6, good[6].half(), TypeError)):
        args = list(good)
        args[i] = x
        with pytest.raises(err):
            bml_b200.verify_drafts(*args)
    for most in (0, -1, 1 << 31):
        with pytest.raises(ValueError):
            bml_b200.verify_drafts(*good, max_path=most)
    with pytest.raises(bml_b200.BmlInvalid):
        bml_b200.verify_drafts(*good[:4], ints([0]), good[5], good[6][:0])


@pytest.mark.parametrize("kind", ["tree", "chain"])
def test_batcher_verifies(cuda, kind):
    """A run of PagedBatcher.verify: lengths and rows are those that commit() with the
    walk's paths leaves in a second batcher."""
    import bml_b200
    rng = np.random.default_rng(11)
    vocab, made = 97, []
    for _ in range(2):
        b = bml_b200.PagedBatcher(2, 4, 2, 64, n_pages=60, page_size=16, max_positions=512, max_requests=5, rope=False)
        for r in "abc":
            b.add(r)
        made.append(b)
    for step in range(5):
        nodes = [int(x) for x in rng.integers(1, 9, 3)]
        if step == 2:
            nodes[1] = 0
        x = batch(nodes, vocab, "f32", True, 50 + step, sharp=0.5)
        new = {r: t if kind == "chain" else x["parents"][sum(nodes[:i]):sum(nodes[:i + 1])] for i, (r, t) in enumerate(zip("abc", nodes)) if t}
        if kind == "chain":
            x["parents"] = [a - 1 for t in nodes for a in range(t)]
        n = sum(nodes)
        rows = [(torch.randn(n, 4, 64, device="cuda").bfloat16(), torch.randn(n, 2, 64, device="cuda").bfloat16()) for _ in range(2)]
        for b in made:
            b.begin(new)
            for layer, (q, k) in enumerate(rows):
                b.step(layer, q.clone(), k, k)
        un = torch.rand(5, device="cuda")
        path, count, token = made[0].verify(x["p"].cuda(), x["q"].cuda(), ints(x["tokens"]), x["u"].cuda(), un)
        paths, at = {}, 0
        for i, (r, t) in enumerate(zip("abc", nodes)):
            s = slice(at, at + t)
            want, nxt = walk(x["p"][s].double().numpy(), x["q"][s].double().numpy(), x["tokens"][s], x["parents"][s], x["u"][s].numpy(),
                             float(un[made[0].place(r)]), 256)
            if t:
                paths[r] = want
            assert count[made[0].place(r)].item() == len(want) and token[made[0].place(r)].item() == nxt
            at += t
        assert count[3:].tolist() == [0, 0] and token[3:].tolist() == [-1, -1]
        made[1].commit(paths)
        for r in "abc":
            assert made[0].length(r) == made[1].length(r)
            for layer in range(2):
                for g, w in zip(made[0].cache(r, layer), made[1].cache(r, layer)):
                    assert torch.equal(g, w)
    with pytest.raises(RuntimeError):
        made[0].verify(x["p"].cuda(), None, ints(x["tokens"]), x["u"].cuda(), un)


@pytest.mark.parametrize("kind", ["tree", "chain"])
def test_batcher_verifies_beside_a_refused_request(cuda, kind):
    """A plan begun without check that refuses a request, for want of pages or of
    places in its table: the request keeps nothing and gets no next token, the
    others get the walk's, and a later step goes on from there."""
    import bml_b200
    b = bml_b200.PagedBatcher(1, 4, 2, 64, n_pages=5, page_size=16, max_positions=48, max_requests=6, rope=False)
    row = lambda n, kv: torch.randn(n, kv, 64, device="cuda").bfloat16()  # noqa: E731
    for r, t in zip("abcd", (30, 15, 2, 0)):             # 2 + 1 + 1 pages of 5
        b.add(r, row(t, 2)[None], row(t, 2)[None])
    nodes = {"a": 12, "b": 4, "c": 20, "d": 60}          # a third page for a, a second for b and c; d's table has 48 places
    before = {r: b.length(r) for r in "abcd"}
    n = sum(nodes.values())
    x = batch(list(nodes.values()), 61, "f32", True, 3, sharp=0.5)
    if kind == "chain":
        x["parents"] = [a - 1 for t in nodes.values() for a in range(t)]
    at, new = 0, {}
    for r, t in nodes.items():
        new[r] = t if kind == "chain" else x["parents"][at:at + t]
        at += t
    plan = b.begin(new, check=False)
    status = plan.status.tolist()
    assert status[:4] == [0, 1, 1, 2], status            # the page that is left is a's
    b.step(0, row(n, 4), row(n, 2), row(n, 2))
    un = torch.rand(6, device="cuda")
    path, count, token = b.verify(x["p"].cuda(), x["q"].cuda(), ints(x["tokens"]), x["u"].cuda(), un)
    want, nxt = walk(x["p"][:12].double().numpy(), x["q"][:12].double().numpy(), x["tokens"][:12], x["parents"][:12], x["u"][:12].numpy(),
                     float(un[0]), 256)
    assert count.tolist() == [len(want), 0, 0, 0, 0, 0] and token.tolist() == [nxt, -1, -1, -1, -1, -1]
    assert path[0, :len(want)].tolist() == want and (path[0, len(want):] == -1).all() and (path[1:] == -1).all()
    assert [b.length(r) for r in "abcd"] == [before["a"] + len(want), before["b"], before["c"], before["d"]]
    # a checked step afterwards keeps everything
    x = batch([1, 1], 61, "f32", True, 4)
    b.begin({"b": 1, "c": 1})
    b.step(0, row(2, 4), row(2, 2), row(2, 2))
    path, count, token = b.verify(x["p"].cuda(), None, ints(x["tokens"]), x["u"].cuda(), un)
    assert count.tolist() == [0, 1, 1, 0, 0, 0] and (token[1:3] >= 0).all()
    assert [b.length(r) for r in "bc"] == [before["b"] + 1, before["c"] + 1]


def test_a_step_and_a_removal_do_not_wait(cuda):
    """begin(check=False), step, verify, commit, remove and compact make no call that
    waits for the GPU, and the lists that the host hands over may go at once.  A
    round before loads the kernels, and more memory is pinned than the round takes,
    since pinning waits."""
    import bml_b200
    b = bml_b200.PagedBatcher(1, 4, 2, 64, n_pages=40, page_size=16, max_positions=128, max_requests=4, rope=False)
    for r in "abc":
        b.add(r)
    n = 14
    x = batch([9, 5], 61, "f32", True, 5)
    p, u, un, tokens = x["p"].cuda(), x["u"].cuda(), torch.rand(4, device="cuda"), ints(x["tokens"])
    q, k = torch.randn(n, 4, 64, device="cuda").bfloat16(), torch.randn(n, 2, 64, device="cuda").bfloat16()
    junk = []

    def steps():
        for kind in ("verify", "commit"):
            b.begin({"a": x["parents"][:9], "b": x["parents"][9:]}, check=False)
            b.step(0, q, k, k)
            if kind == "verify":
                got = b.verify(p, None, tokens, u, un)
            else:
                b.commit({"a": [0, 2, 5], "b": []})
            junk.extend(torch.full((size,), -7, dtype=torch.int32, pin_memory=True) for size in (2, 4, 5, 9, 14, 16))
        b.remove("c")
        b.compact()
        return got

    steps()
    junk.extend(torch.empty(size, dtype=torch.int32, pin_memory=True) for size in (2, 4, 8, 16, 32) for _ in range(40))
    del junk[:]
    b.add("c")
    for r in "ab":
        b.truncate(r, 0)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        torch.cuda._sleep(1_000_000_000)                 # the copies lie behind half a second of work
        path, count, token = steps()
        busy = not torch.cuda.current_stream().query()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert busy
    want = [walk(x["p"][s].double().numpy(), None, x["tokens"][s], x["parents"][s], x["u"][s].numpy(), float(un[i]), 256)
            for i, s in enumerate((slice(0, 9), slice(9, 14)))]
    assert count.tolist() == [len(want[0][0]), len(want[1][0]), 0, 0] and token.tolist() == [want[0][1], want[1][1], -1, -1]
    assert b.length("a") == len(want[0][0]) + 3 and b.length("b") == len(want[1][0])
    assert b.active == ["a", "b"] and int(b.used) == int(b.owned.sum())


def test_a_batchers_host_state_is_not_captured(cuda):
    """The lists of a plan, a commit or a removal lie in host memory that is used again:
    such a call in a graph is refused and changes nothing; the layers' calls may be captured."""
    import bml_b200
    b = bml_b200.PagedBatcher(1, 4, 2, 64, n_pages=8, page_size=16, max_positions=64, max_requests=2, rope=False)
    b.add("a")
    q, k = torch.randn(2, 4, 64, device="cuda").bfloat16(), torch.randn(2, 2, 64, device="cuda").bfloat16()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        for call in (lambda: b.begin({"a": 2}, check=False), lambda: b.remove("a"), lambda: b.fork("a", "b")):
            with pytest.raises(RuntimeError, match="captured"):
                call()
        junk = q + 1                                     # a graph that holds something
    assert b.active == ["a"]
    b.begin({"a": 2})
    b.step(0, q, k, k)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = b.step(0, q, k, k)
        with pytest.raises(RuntimeError, match="captured"):
            b.commit()
    g.replay()
    want = b.step(0, q, k, k)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    b.commit()
    assert b.length("a") == 2
    del g, junk
