"""GPU tests of arguments of the paged wrappers at the ends of their ranges."""
import pytest
import torch

from test_paged_gpu import ints

pytestmark = pytest.mark.gpu


def test_counts_past_32_bits_are_refused(cuda):
    """Not taken modulo 2^32."""
    import bml_b200
    one = ints([1])
    table, free = ints([[-1, -1]]), ints([0, 1])
    for page, n in ((2 ** 32 + 16, 1), (16, 2 ** 32 + 1), (-2 ** 32 + 16, 1), (16, 2 ** 31)):
        with pytest.raises(ValueError):
            bml_b200.page_plan(one, one, ints([1]), table, free, ints([0]), page, n)
    with pytest.raises(bml_b200.BmlInvalid):
        bml_b200.page_plan(one, one, ints([1]), table, free, ints([0]), 0, 1)
    assert table.tolist() == [[-1, -1]]


def test_commit_none_keeps_all(cuda):
    """A path of None is a request that is not named, [] one that keeps nothing."""
    import bml_b200
    b = bml_b200.PagedBatcher(1, 4, 2, 64, n_pages=8, page_size=16, max_positions=64, max_requests=3)
    for r in "abc":
        b.add(r)
    b.begin({"a": 3, "b": 4, "c": 5})
    q, kv = (torch.zeros(12, h, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
    b.step(0, q, kv, kv)
    b.commit({"a": None, "b": []})
    assert [b.length(r) for r in "abc"] == [3, 0, 5]
