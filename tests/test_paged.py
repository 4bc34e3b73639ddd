"""Refusals of the paged-cache entry points, on the CPU: the C functions check
their arguments before anything is launched, the Python ones before that."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from bml_b200 import build
    build.build()
    import bml_b200._lib as lib
    return lib


A = 1 << 20  # an aligned address that no refused call reads


def plan(lib, **kw):
    a = dict(lens=A, n_new=A, owned=A, n=2, free_pages=A, n_free=4, free_used=A, page_size=16, max_pages=8,
             block_table=A, parents=A, n_tokens=4, n_words=1, node_start=A, kv_lens=A, owned_out=A + 64,
             free_used_out=A + 128, slots=A, positions=A, mask=A, status=A, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.bml_paged_plan(*a.values())


def append(lib, **kw):
    a = dict(q=A, k=A, v=A, src=0, slots=A, positions=A, n_tokens=4, n_heads=4, n_kv=2, head_dim=64, theta=10000.0,
             q_out=A, k_pool=A, v_pool=A, kv=2, n_rows=64, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.bml_paged_append(*a.values())


def attend(lib, **kw):
    a = dict(q=A, q_dtype=2, n_tokens=4, n_heads=4, n_kv=2, head_dim=64, k=A, v=A, kv=2, n_pages=4, page_size=16,
             table=A, max_pages=8, kv_lens=A, node_start=A, n_seqs=2, mask=A, n_words=1, scale=-1.0, out=2 * A, ws=A,
             ws_bytes=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.bml_attn_tree(*a.values())


def commit(lib, **kw):
    a = dict(k=A, v=A, n_layers=2, n_pages=4, page_size=16, n_kv=2, head_dim=64, kv=2, table=A, max_pages=8, lens=A,
             kv_lens=A, node_start=A, n=2, path=A, max_path=4, n_accept=A, lens_out=2 * A, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.bml_paged_commit(*a.values())


@pytest.mark.parametrize("call,bad", [
    (plan, dict(n=0)), (plan, dict(n=4097)), (plan, dict(page_size=8)), (plan, dict(page_size=24)),
    (plan, dict(page_size=2048)), (plan, dict(max_pages=0)), (plan, dict(max_pages=1 << 27)), (plan, dict(lens=None)),
    (plan, dict(owned=A + 2)), (plan, dict(owned_out=A)), (plan, dict(free_used_out=A)), (plan, dict(n_words=0)),
    (plan, dict(n_words=5)), (plan, dict(mask=None)), (plan, dict(mask=A + 4)), (plan, dict(slots=A + 4)),
    (plan, dict(free_pages=None)), (plan, dict(status=None)), (plan, dict(n_tokens=1 << 31)),
    (append, dict(head_dim=63)), (append, dict(head_dim=0)), (append, dict(n_kv=0)), (append, dict(q=None)),
    (append, dict(q_out=None)), (append, dict(src=7)), (append, dict(kv=-1)), (append, dict(k=None)),
    (append, dict(slots=None)), (append, dict(slots=A + 4)), (append, dict(k=A + 4)), (append, dict(k_pool=A + 2)),
    (append, dict(theta=0.0)), (append, dict(theta=float("inf"))), (append, dict(n_heads=0)),
    (append, dict(n_rows=1 << 31)), (append, dict(q_out=A + 1024)),
    (attend, dict(n_heads=3)), (attend, dict(n_kv=0)), (attend, dict(n_seqs=0)), (attend, dict(n_pages=0)),
    (attend, dict(page_size=12)), (attend, dict(n_pages=1 << 27)), (attend, dict(max_pages=0)),
    (attend, dict(n_words=5)), (attend, dict(n_words=0)), (attend, dict(scale=float("nan"))),
    (attend, dict(scale=float("inf"))), (attend, dict(table=None)), (attend, dict(kv_lens=A + 1)),
    (attend, dict(q=None)), (attend, dict(q=A + 8)), (attend, dict(out=A)), (attend, dict(out=A + 256)),
    (attend, dict(ws=None)), (attend, dict(ws_bytes=1 << 20)), (attend, dict(mask=A + 4)), (attend, dict(kv=9)),
    (commit, dict(n_layers=0)), (commit, dict(n_layers=32768)), (commit, dict(n=0)), (commit, dict(max_path=0)),
    (commit, dict(page_size=17)), (commit, dict(lens_out=A)), (commit, dict(path=None)), (commit, dict(k=None)),
    (commit, dict(kv=3)), (commit, dict(head_dim=0)), (commit, dict(n_pages=1 << 28)),
])
def test_invalid_arguments(L, call, bad):
    assert call(L.lib(), **bad) == L.BML_E_INVALID
    assert L.last_error()


B = 1 << 24
APART = {  # (call, arrays it reads, arrays it writes)
    plan: (("lens", "n_new", "owned", "free_pages", "free_used", "parents"),
           ("node_start", "kv_lens", "owned_out", "free_used_out", "status", "slots", "positions", "mask", "block_table")),
    commit: (("lens", "kv_lens", "node_start", "n_accept", "path", "table"), ("lens_out",)),
}


@pytest.mark.parametrize("call,read,written", [(c, r, w) for c, (rs, ws) in APART.items() for r in rs for w in ws])
def test_results_have_buffers_of_their_own(L, call, read, written):
    """An array that a call both reads and writes, or one that ends inside
    another, is refused: its CTAs do not wait for one another."""
    names = APART[call][0] + APART[call][1]
    apart = {n: B + 4096 * i for i, n in enumerate(names)}
    before = {"free_used_out": 0, "slots": 8, "mask": 8}.get(written, 4)
    for same in (apart[read], apart[read] - before):
        assert call(L.lib(), **{**apart, written: same}) == L.BML_E_INVALID
        assert "own" in L.last_error()


def test_unsupported(L):
    lib = L.lib()
    assert append(lib, theta=1e-6) == L.BML_E_UNSUPPORTED
    assert attend(lib, scale=3e38) == L.BML_E_INVALID         # not finite in units of log2
    assert attend(lib, head_dim=96) == L.BML_E_UNSUPPORTED
    assert attend(lib, q_dtype=1) == L.BML_E_UNSUPPORTED      # f16 queries, bf16 pages
    assert attend(lib, q_dtype=2, kv=0) == L.BML_E_UNSUPPORTED
    assert append(lib, head_dim=2048) == L.BML_E_UNSUPPORTED
    n = C.c_size_t()
    assert lib.bml_attn_tree_workspace_size(96, 0, C.byref(n)) == L.BML_E_UNSUPPORTED
    assert lib.bml_attn_tree_workspace_size(64, 0, None) == L.BML_E_INVALID


def test_nothing_to_do(L):
    lib = L.lib()
    assert append(lib, n_tokens=0) == L.BML_OK
    assert attend(lib, n_tokens=0) == L.BML_OK


def test_workspace_size(L):
    n = C.c_size_t()
    assert L.lib().bml_attn_tree_workspace_size(128, 0, C.byref(n)) == L.BML_OK
    assert 0 < n.value < 1 << 27


def test_python_refusals(L):
    """CPU tensors are refused by name before the library is reached."""
    import bml_b200
    i, x = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, 64)
    with pytest.raises(ValueError, match="lens"):
        bml_b200.page_plan(i, i, i, i, i, i, 16, 4)
    with pytest.raises(ValueError, match="k must"):
        bml_b200.paged_append(x, x, x, i, i, x, x)
    with pytest.raises(ValueError, match="q must"):
        bml_b200.tree_attention(x, x, x, i, i, i)
    with pytest.raises(ValueError, match="k_pool"):
        bml_b200.paged_commit(x, x, i, i, i, i, i, i)
