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
