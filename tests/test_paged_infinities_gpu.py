"""GPU tests of tree_attention: infinities that a row sees, and the largest
finite values.  Cases and tolerances as in test_paged_gpu.py."""
import numpy as np
import pytest
import torch

from test_paged_gpu import TYPES, Paged, chain, check, pack, tol
from test_paged_masked_gpu import put, widen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nodes", [[1, 1, 1], [3, 2, 5], [40, 40, 3], [64, 130, 64]])
@pytest.mark.parametrize("wide", [False, True])
def test_infinities_that_are_seen(cuda, qt, ct, d, nodes, wide):
    """An infinity in a V row that a row sees is one in those columns, whatever
    its weight and whichever tile it lies in, two of different sign are NaN; an
    infinite score of -inf weighs nothing, one of +inf makes the row NaN."""
    import bml_b200
    lens, page = [300, 517, 2000], 16
    inf = float("inf")
    for where in (0, 17, 130, 299):
        c = Paged(lens, nodes, 8, 2, d, page, qt, ct, seed=60)
        if wide:
            widen(c, page)
        at = [int(c.table[i, where // page]) for i in range(3)]
        c.v[at[0], where % page, 0, 7] = inf
        c.v[at[0], where % page, 1, 8] = -inf
        two = where + 1 if where % page < page - 1 else where - 1   # on the same page
        c.v[at[1], where % page, 0, 3], c.v[at[1], two % page, 0, 3] = inf, -inf
        c.k[at[2], where % page, 0, 5] = inf
        c.k[at[2], two % page, 0, 6] = -inf
        c.ks[2][where, 0, 5], c.ks[2][two, 0, 6] = inf, -inf
        got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start)
        s = c.start.tolist()
        a, b, z = got[:s[1]], got[s[1]:s[2]], got[s[2]:]
        assert torch.isposinf(a[:, :4, 7]).all() and torch.isneginf(a[:, 4:, 8]).all()
        assert torch.isnan(b[:, :4, 3]).all()
        # a score is +inf where q and k have the same sign there: those rows are NaN, the others finite
        q = c.q[s[2]:, :4].float()
        plus = (q[..., 5] > 0) | (q[..., 6] < 0)
        assert torch.equal(torch.isnan(z[:, :4]).all(-1), plus) and torch.equal(torch.isnan(z[:, :4]).any(-1), plus)
        # and everything else is what it is without them
        a[:, :4, 7] = a[:, 4:, 8] = b[:, :4, 3] = 0
        z[:, :4] = 0
        for i in range(2):
            want, ab, bmax = c.want(i, chain(nodes[i], lens[i]))
            have = (a, b)[i].double()
            if i == 0:
                want[:, :4, 7] = want[:, 4:, 8] = 0
            else:
                want[:, :4, 3] = 0
            assert torch.isfinite(have).all()
            assert ((have - want).abs() <= tol(qt, want, ab, bmax)).all()
        rest = c.want(2, chain(nodes[2], lens[2]))
        have = z[:, 4:].double()
        assert ((have - rest[0][:, 4:]).abs() <= tol(qt, rest[0], rest[1], rest[2])[:, 4:]).all()


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("nodes", [[1, 1], [6, 3], [50, 33]])
def test_weightless_infinities(cuda, qt, ct, nodes):
    """A position whose weight is too small for 32 bits, with an infinity in V:
    weights are positive, so the column is infinite; and a request cut over many
    CTAs, with the infinity in the part of the smaller scores."""
    import bml_b200
    d, page = 64, 16
    c = Paged([90, 30000], nodes, 4, 2, d, page, qt, ct, seed=61)
    c.q.abs_()
    for i, low in ((0, 40), (1, 500)):
        pos = torch.arange(low, device="cuda")
        at = c.table[i].long()[pos // page]
        c.ks[i][:low] = -c.ks[i][:low].abs() * 4
        c.k[at, pos % page] = c.ks[i][:low]
        c.v[int(c.table[i, 0]), 3, 1, 9] = float("inf")
        c.vs[i][3, 1, 9] = 0.0
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, scale=1.0)
    assert torch.isposinf(got[:, 2:, 9]).all()
    got[:, 2:, 9] = 0
    for i in range(2):
        want, ab, bmax = c.want(i, chain(nodes[i], c.lens[i]), 1.0)
        s = c.start.tolist()
        want[:, 2:, 9] = 0
        assert ((got[s[i]:s[i + 1]].double() - want).abs() <= tol(qt, want, ab, bmax)).all()


@pytest.mark.parametrize("nodes", [[1, 1], [4, 6], [40, 33]])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_largest_f32_values(cuda, nodes, wide, d):
    """32-bit pages with values up to the largest finite f32: in V rows that are
    seen with weights that sum to 1 (so un-normalised sums stay in range only for
    small weights: one position holds them), in masked nodes, and in K beside a
    query of zeros there."""
    import bml_b200
    page, big = 16, torch.finfo(torch.float32).max
    lens = [150, 40]
    c = Paged(lens, nodes, 8, 2, d, page, "f32", "f32", seed=62)
    if wide:
        widen(c, page)
    # a small score, so that its weight, at most 2^-8 of the largest, keeps the sum in range
    c.q.abs_()
    for i, pos in ((0, 70), (1, 33)):
        put(c, i, pos, page, k=-3.0, v=big)
    c.q[:, :, 11] = 0.0
    at = int(c.table[0, 20 // page])
    c.k[at, 20 % page, :, 11] = big
    c.ks[0][20, :, 11] = big
    masks = [np.tril(np.ones((t, t), bool)) for t in nodes]
    if nodes[0] > 1:
        for i in range(2):
            masks[i][:, 1] = False
            put(c, i, lens[i] + 1, page, v=-big)
    sees = [np.concatenate([np.ones((t, p), bool), m], 1) for t, p, m in zip(nodes, lens, masks)]
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, mask=pack(masks, 1))
    check(c, got, sees, "f32")
