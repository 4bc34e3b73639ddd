"""GPU tests of batches of which most places are idle, or hold single tokens beside
a wide draft.  Cases and tolerances as in test_paged_gpu.py."""
import numpy as np
import pytest
import torch

from test_paged_gpu import TYPES, Paged, check, mask_of, pack, random_parents

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_hints(cuda, qt, ct, d):
    """Results are right with every hint, right or wrong, on either way of the wrapper."""
    import bml_b200
    rng = np.random.default_rng(80)
    nodes = [0] * 20 + [64, 1, 1, 0, 9, 100] + [0] * 10
    lens = [int(x) for x in rng.integers(0, 600, len(nodes))]
    c = Paged(lens, nodes, 8, 2, d, 16, qt, ct, seed=81)
    masks = [mask_of(random_parents(rng, t)) for t in nodes]
    sees = [np.concatenate([np.ones((t, p), bool), m.reshape(t, t)], 1) for t, p, m in zip(nodes, lens, masks)]
    m = pack(masks, 2)
    args = (c.q, c.k, c.v, c.table, c.kv_lens, c.start)
    for n_live, max_new in ((0, 0), (5, 100), (1, 1), (0, 100), (5, 0), (10 ** 6, 10 ** 6)):
        got = bml_b200.tree_attention(*args, mask=m, n_live=n_live, max_new=max_new)
        check(c, got, sees, qt)
        own = bml_b200.tree_attention(*args, mask=m, n_live=n_live, max_new=max_new, out=torch.empty_like(c.q))
        assert torch.equal(own, got)
    for bad in (dict(n_live=-1), dict(max_new=-2)):
        with pytest.raises(ValueError):
            bml_b200.tree_attention(*args, mask=m, **bad)


def test_batcher_says_how_many(cuda, monkeypatch):
    """PagedBatcher hands on how many places have new tokens, and the most of one."""
    import bml_b200
    import bml_b200.paged as P
    b = bml_b200.PagedBatcher(1, 8, 2, 64, n_pages=64, page_size=16, max_positions=256)
    for r in "abc":
        b.add(r)
    said = []
    real = P.tree_attention
    monkeypatch.setattr(P, "tree_attention", lambda *a, **kw: said.append((kw["n_live"], kw["max_new"])) or real(*a, **kw))
    for new in ({"a": 5, "c": [-1, 0, 1, 1, 0, 2, 3]}, {"b": 1}, {}, {"a": 0, "b": 2, "c": 1}):
        b.begin(new)
        n = sum(x if isinstance(x, int) else len(x) for x in new.values())
        q, k, v = (torch.randn(n, h, 64, device="cuda").bfloat16() for h in (8, 2, 2))
        b.step(0, q, k, v)
        b.commit()
    assert said == [(2, 7), (1, 1), (0, 0), (2, 2)]
