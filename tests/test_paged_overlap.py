"""Refusals of arrays that overlap, on the CPU: nothing here is launched.  A call's
CTAs do not wait for one another, so that what one writes another may not have
read yet."""
import pytest

from test_paged import L, append, attend, commit, plan  # noqa: F401 (L: the fixture)

B = 1 << 30  # far from everything else
SPAN = 1 << 25
APPEND = {n: B + SPAN * i for i, n in enumerate(("q", "k", "v", "slots", "positions", "q_out", "k_pool", "v_pool"))}
ATTEND = {n: B + SPAN * i for i, n in enumerate(("q", "k", "v", "table", "kv_lens", "node_start", "mask", "out", "ws"))}
PLAN = {n: B + SPAN * i for i, n in enumerate(("lens", "n_new", "owned", "free_pages", "free_used", "parents", "node_start", "kv_lens",
                                               "owned_out", "free_used_out", "status", "slots", "positions", "mask", "block_table"))}


@pytest.mark.parametrize("written,other", [(w, o) for w in ("q_out", "k_pool", "v_pool") for o in APPEND if o != w])
def test_append(L, written, other):
    """The pools and q_out on one another, and on what is read."""
    if (written, other) == ("q_out", "q"):
        pytest.skip("in place")
    for at in (APPEND[other], APPEND[other] + 16, APPEND[other] - 16):
        if other in ("slots", "positions") and at > APPEND[other]:
            continue  # behind the 16 bytes of positions
        assert append(L.lib(), **{**APPEND, written: at}) == L.BML_E_INVALID
        assert "overlap" in L.last_error()


@pytest.mark.parametrize("written,other", [(w, o) for w in ("out", "ws") for o in ATTEND if o != w])
def test_attend(L, written, other):
    for at in (ATTEND[other], ATTEND[other] - 16):
        assert attend(L.lib(), **{**ATTEND, written: at}) == L.BML_E_INVALID
        assert "overlap" in L.last_error()


def test_commit_of_one_pool(L):
    """Both CTAs of a row would move it: the second reads what the first has written."""
    apart = {n: B + 4096 * i for i, n in enumerate(("table", "lens", "kv_lens", "node_start", "path", "n_accept", "lens_out"))}
    pool = 2 * 4 * 16 * 2 * 64 * 2
    for v in (0, pool - 16, 16 - pool):
        assert commit(L.lib(), **apart, k=B + SPAN, v=B + SPAN + v) == L.BML_E_INVALID
        assert "overlap" in L.last_error()


WRITTEN = ("node_start", "kv_lens", "owned_out", "free_used_out", "status", "slots", "positions", "mask", "block_table")


@pytest.mark.parametrize("a,b", [(a, b) for i, a in enumerate(WRITTEN) for b in WRITTEN[i + 1:]])
def test_plan_results_on_one_another(L, a, b):
    assert plan(L.lib(), **{**PLAN, b: PLAN[a]}) == L.BML_E_INVALID
    assert "overlap" in L.last_error()
