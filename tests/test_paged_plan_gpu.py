"""GPU tests of page_plan near the most requests, and with its arguments chosen
apart from one another."""
import os
import subprocess
import sys

import numpy as np
import pytest

from test_paged_gpu import ints, plan_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [4085, 4086, 4095])
def test_plan_near_the_most_requests(cuda, n):
    """In a process of its own: a kernel's allowance of shared memory stays once
    a larger call has raised it."""
    run_alone(f"for m in ({n}, 4096):\n  for tree in (False, True): plan_of_many(m, tree, 64, 1, 0, 7)")


def run_alone(call):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", f"import sys; sys.path[:0] = [{root!r}, {root + '/tests'!r}]\n"
                        f"from test_paged_plan_gpu import *\n{call}"], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0, r.stderr[-2000:]


def plan_of_many(n, tree, page, words, extra, seed):
    """A plan of n requests, some of them bad, against the plain planner."""
    import bml_b200
    rng = np.random.default_rng(seed)
    hi = 64 * words if tree else 300
    lens = rng.integers(0, 500, n)
    new = rng.integers(0, hi + 1, n) * (rng.random(n) < 0.8)
    if n > 1000:
        new //= 8
    owned = -(-lens // page) + rng.integers(0, 2, n)
    if n > 30:
        lens[3], new[5], owned[7] = -1, -4, -2
        lens[11] = 100000
        new[17] = 64 * words + 1
    mp = -(-2000 // page)
    need = int(np.maximum(0, -(-(lens + new) // page) - owned)[owned >= 0].sum())
    used = int(rng.integers(0, 10))
    free = rng.permutation(max(1, used + (need if seed % 3 else need // 2)))
    table = rng.integers(0, 1000, (n, mp))
    n_tokens = max(0, int(np.maximum(new, 0).sum()) + extra)
    parents = rng.integers(-2, 70, n_tokens) if tree else None
    args = [ints(lens), ints(new), ints(owned), ints(table), ints(free), ints([used])]
    p = bml_b200.page_plan(*args, page, n_tokens, parents=ints(parents) if tree else None, n_words=words)
    w = plan_reference(lens.tolist(), new.tolist(), owned.tolist(), table, free.tolist(), used, page, n_tokens,
                       parents.tolist() if tree else None, words)
    assert np.array_equal(args[3].cpu().numpy(), w[0])
    for got, want in ((p.node_start, w[1]), (p.kv_lens, w[2]), (p.owned, w[3]), (p.free_used, [w[4]]),
                      (p.slots, w[5]), (p.positions, w[6]), (p.status, w[7])):
        assert got.tolist() == want
    if tree and n_tokens:
        assert np.array_equal(p.mask.cpu().numpy().view(np.uint64), np.array(w[8], np.uint64))


@pytest.mark.parametrize("n", [1, 3, 40, 257, 1000])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("page,words,extra", [(16, 4, -20), (32, 1, 5), (1024, 2, 0), (64, 1, -20), (16, 2, 5)])
def test_plans(cuda, n, tree, page, words, extra):
    """Requests, drafts, pages, mask words and the token rows' count chosen apart."""
    plan_of_many(n, tree, page, words, extra, n + page)
