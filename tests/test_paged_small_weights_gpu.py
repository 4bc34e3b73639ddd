"""GPU tests of tree_attention: columns in which the heavy positions hold zeros, so
that only small weights count.  Cases and tolerances as in test_paged_gpu.py: of a
column, relative to its own sum of p |v|.

32-bit queries over f16 pages split a weight into two f16 terms, the second kept
2^12 times as large.  A weight on its way is at most 2^15, and the largest of a row
at least 2^7, times what it is relative to that largest: half of the second term's
smallest step, 2^-25, is 2^-37 of that, so 2^-44 of the largest weight, which is at
most 1.  A column's sum may be off by as much times the sum of |v|."""
import pytest
import torch

from test_paged_gpu import TYPES, Paged, chain, tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nodes", [[1, 1], [3, 2], [7, 20], [40, 64]])
@pytest.mark.parametrize("scale", [0.02, 0.1, 0.3, 1.0])
def test_columns_of_small_weights(cuda, qt, ct, d, nodes, scale):
    import bml_b200
    lens = [90, 700]
    c = Paged(lens, nodes, 8, 2, d, 16, qt, ct, seed=90)
    for i in range(2):
        pos = torch.arange(lens[i], device="cuda")
        at = c.table[i].long()[pos // 16]
        # the heads' heaviest positions (of any row) have zeros in the even columns
        s = torch.einsum("thd,lhd->htl", c.q[int(c.start[i]):int(c.start[i + 1])].float(),
                         c.ks[i][:lens[i]].float().repeat_interleave(4, 1)).amax(1)
        heavy = torch.zeros(lens[i], 2, dtype=torch.bool, device="cuda")
        for h in range(2):
            heavy[s[4 * h:4 * h + 4].amax(0).topk(min(lens[i] // 2, 60)).indices, h] = True
        v = c.vs[i][:lens[i]]
        v[..., ::2] = torch.where(heavy[..., None], torch.zeros_like(v[..., ::2]), v[..., ::2])
        c.v[at, pos % 16] = v
        # and so have the nodes
        node = torch.arange(lens[i], lens[i] + nodes[i], device="cuda")
        c.vs[i][lens[i]:, :, ::2] = 0
        c.v[c.table[i].long()[node // 16], node % 16] = c.vs[i][lens[i]:]
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, scale=scale)
    for i in range(2):
        a, b = int(c.start[i]), int(c.start[i + 1])
        want, ab, bmax = c.want(i, chain(nodes[i], lens[i]), scale)
        lim = tol(qt, want, ab, bmax)
        if (qt, ct) == ("f32", "f16"):
            lim = lim + 2.0 ** -44 * c.vs[i].double().abs().sum(0).repeat_interleave(4, 0)
        assert ((got[a:b].double() - want).abs() <= lim).all()
