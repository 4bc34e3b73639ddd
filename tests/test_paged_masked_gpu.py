"""GPU tests of tree_attention: large finite values in masked places.  Cases and
tolerances as in test_paged_gpu.py."""
import numpy as np
import pytest
import torch

from test_paged_gpu import TYPES, Paged, check, mask_of, pack, random_parents

pytestmark = pytest.mark.gpu


def widen(c, page, positions=16384):
    """Tables far wider than the requests, which the kernels for much work take."""
    more = torch.full((c.table.shape[0], positions // page), -1, dtype=torch.int32, device="cuda")
    c.table = torch.cat([c.table, more], 1).contiguous()


def put(c, i, pos, page, k=None, v=None):
    """One value for a whole K or V row of request i (in the pages and in the formula's copy)."""
    at = int(c.table[i, pos // page])
    if k is not None:
        c.k[at, pos % page] = k
        c.ks[i][pos] = k
    if v is not None:
        c.v[at, pos % page] = v
        c.vs[i][pos] = v


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("wide", [False, True])
def test_large_values_in_masked_nodes(cuda, qt, ct, d, wide):
    """Finite V values near the type's largest in nodes that a row does not see,
    at every place of a 16-position block, add nothing to it."""
    import bml_b200
    lens, nodes, page = [0, 203, 40, 300], [33, 40, 64, 1], 16
    c = Paged(lens, nodes, 16, 2, d, page, qt, ct, seed=50 + d)
    if wide:
        widen(c, page)
    rng = np.random.default_rng(5)
    big = {"bf16": 3.38e38, "f16": 65504.0, "f32": 1e38}[ct]
    masks = [mask_of(random_parents(rng, t)) for t in nodes]
    for i, t in enumerate(nodes[:3]):
        for node in range(t // 2, t - 1):            # seen by nobody
            masks[i][:, node] = False
            put(c, i, lens[i] + node, page, v=big if node % 2 else -big)
    sees = [np.concatenate([np.ones((t, p), bool), m.reshape(t, t)], 1) for t, p, m in zip(nodes, lens, masks)]
    got = bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start, mask=pack(masks, 1))
    check(c, got, sees, qt)
