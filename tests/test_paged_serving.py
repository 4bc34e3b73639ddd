"""Refusals of chunk_attention, verify_drafts and the pages' calls on the CPU: the C
functions check their arguments before anything is launched, the Python ones
before that."""
import ctypes as C

import pytest
import torch

from test_paged import L  # noqa: F401 (the fixture)

A, SPAN = 1 << 30, 1 << 26


def apart(*names):
    return {n: A + SPAN * i for i, n in enumerate(names)}


def caller(fn, order, arrays, **rest):
    base = {**apart(*arrays), **rest, "stream": None}

    def call(lib, **kw):
        assert set(kw) <= set(base)
        a = {**base, **kw}
        return getattr(lib, fn)(*(a[n] for n in order.split()))
    call.arrays = arrays
    call.fn = fn
    return call


chunk = caller("bml_attn_chunk", "q qt n_tokens n_heads n_kv d k v kt n_pages page table max_pages kv_lens start n scale out ws "
               "ws_bytes live most stream", ("q", "k", "v", "table", "kv_lens", "start", "out", "ws"), qt=2, n_tokens=4, n_heads=4, n_kv=2,
               d=64, kt=2, n_pages=4, page=16, max_pages=8, n=2, scale=-1.0, ws_bytes=1 << 40, live=0, most=0)
verify = caller("bml_verify_drafts", "p q dt vocab tok par n_tokens start n u un max_path path count next stream",
                ("p", "q", "tok", "par", "start", "u", "un", "path", "count", "next"), dt=0, vocab=100, n_tokens=6, n=2, max_path=4)
fork = caller("bml_page_fork", "k v layers n_pages page n_kv d dt src dst m lens owned n table max_pages shared free n_free used lens2 "
              "owned2 shared2 used2 status stream", ("k", "v", "src", "dst", "lens", "owned", "table", "shared", "free", "used", "lens2",
                                                     "owned2", "shared2", "used2", "status"),
              layers=2, n_pages=4, page=16, n_kv=2, d=64, dt=2, m=2, n=3, max_pages=8, n_free=4)
free = caller("bml_page_free", "keep lens owned n table max_pages page shared n_pages free n_free used lens2 owned2 shared2 free2 used2 "
              "status ws ws_bytes stream", ("keep", "lens", "owned", "table", "shared", "free", "used", "lens2", "owned2", "shared2", "free2",
                                            "used2", "status", "ws"), n=3, max_pages=8, page=16, n_pages=4, n_free=4, ws_bytes=4100)
compact = caller("bml_page_compact", "k v layers n_pages page n_kv d dt owned n table max_pages shared table2 shared2 free2 used2 ws "
                 "ws_bytes stream", ("k", "v", "owned", "table", "shared", "table2", "shared2", "free2", "used2", "ws"),
                 layers=2, n_pages=4, page=16, n_kv=2, d=64, dt=2, n=3, max_pages=8, ws_bytes=52)
WRITTEN = {chunk: ("out", "ws"), verify: ("path", "count", "next"),
           fork: ("k", "v", "table", "lens2", "owned2", "shared2", "used2", "status"),
           free: ("lens2", "owned2", "shared2", "free2", "used2", "status", "ws"),
           compact: ("k", "v", "table2", "shared2", "free2", "used2", "ws")}


@pytest.mark.parametrize("call,bad", [
    (chunk, dict(n_heads=3)), (chunk, dict(n_kv=0)), (chunk, dict(n=0)), (chunk, dict(n_pages=0)), (chunk, dict(page=12)),
    (chunk, dict(n_pages=1 << 27)), (chunk, dict(max_pages=0)), (chunk, dict(scale=float("nan"))), (chunk, dict(scale=float("inf"))),
    (chunk, dict(table=None)), (chunk, dict(kv_lens=A + 1)), (chunk, dict(q=None)), (chunk, dict(q=A + 8)),
    (chunk, dict(ws=None)), (chunk, dict(ws_bytes=1 << 20)), (chunk, dict(kt=9)), (chunk, dict(n_tokens=1 << 31)),
    (verify, dict(dt=3)), (verify, dict(vocab=0)), (verify, dict(vocab=1 << 31)), (verify, dict(n=0)), (verify, dict(n=1 << 23)),
    (verify, dict(max_path=0)), (verify, dict(max_path=1 << 31)), (verify, dict(n_tokens=1 << 31)), (verify, dict(p=None)),
    (verify, dict(p=A + 2)), (verify, dict(q=A + 2)), (verify, dict(tok=None)), (verify, dict(par=A + 1)), (verify, dict(start=None)),
    (verify, dict(u=None)), (verify, dict(un=None)), (verify, dict(path=None)), (verify, dict(count=A + 2)), (verify, dict(next=None)),
    (fork, dict(n=0)), (fork, dict(n=4097)), (fork, dict(m=4097)), (fork, dict(page=24)), (fork, dict(max_pages=0)), (fork, dict(dt=5)),
    (fork, dict(layers=0)), (fork, dict(layers=32768)), (fork, dict(n_pages=0)), (fork, dict(n_kv=0)), (fork, dict(d=0)),
    (fork, dict(n_pages=1 << 27)), (fork, dict(n_kv=1 << 20, d=1 << 12)), (fork, dict(k=None)), (fork, dict(v=A + 2)), (fork, dict(src=None)),
    (fork, dict(status=None)), (fork, dict(free=None)), (fork, dict(lens2=None)), (fork, dict(n_free=1 << 31)), (fork, dict(shared=A + 1)),
    (free, dict(n=0)), (free, dict(n=4097)), (free, dict(page=0)), (free, dict(max_pages=1 << 27)), (free, dict(n_pages=0)),
    (free, dict(n_pages=1 << 27)), (free, dict(keep=None)), (free, dict(free=None)), (free, dict(free2=None)), (free, dict(n_free=1 << 31)),
    (free, dict(status=A + 2)), (free, dict(ws=None)), (free, dict(ws=A + 2)), (free, dict(ws_bytes=4099)), (compact, dict(n=0)), (compact, dict(n=4097)), (compact, dict(page=17)), (compact, dict(n_pages=0)),
    (compact, dict(dt=-1)), (compact, dict(owned=None)), (compact, dict(ws=None)), (compact, dict(ws_bytes=51)), (compact, dict(k=None)),
    (compact, dict(d=1 << 30)), (compact, dict(table2=A + 3)),
])
def test_invalid_arguments(L, call, bad):
    assert call(L.lib(), **bad) == L.BML_E_INVALID
    assert call.fn in L.last_error()


@pytest.mark.parametrize("call,written,other", [(c, w, o) for c, ws in WRITTEN.items() for w in ws for o in c.arrays if o != w])
def test_overlaps(L, call, written, other):
    """What a call writes on what it reads or writes besides."""
    base = apart(*call.arrays)
    for at in (base[other], base[other] + 4 if call is not chunk and other in ("k", "v", "p", "q", "table") else base[other]):
        assert call(L.lib(), **{written: at}) == L.BML_E_INVALID
        assert "overlap" in L.last_error()


def test_unsupported_and_nothing_to_do(L):
    lib = L.lib()
    assert chunk(lib, d=96) == L.BML_E_UNSUPPORTED
    assert chunk(lib, qt=1) == L.BML_E_UNSUPPORTED       # f16 queries, bf16 pages
    assert chunk(lib, n_tokens=0) == L.BML_OK
    n, m = C.c_size_t(), C.c_size_t()
    assert lib.bml_attn_chunk_workspace_size(96, 1, 1, 0, C.byref(n)) == L.BML_E_UNSUPPORTED
    assert lib.bml_attn_chunk_workspace_size(64, 1, 1, 0, None) == L.BML_E_INVALID
    assert lib.bml_attn_chunk_workspace_size(64, 5000, 7, 0, C.byref(n)) == L.BML_OK
    assert lib.bml_attn_tree_workspace_size(64, 0, C.byref(m)) == L.BML_OK
    assert m.value < n.value < 4 * m.value + (1 << 17)   # the results of a long line's pieces, of up to four passes over it
    assert lib.bml_attn_chunk_workspace_size(64, 1000, 7, 0, C.byref(n)) == L.BML_OK
    assert m.value < n.value < m.value + (1 << 17)       # of one pass
    assert chunk(lib, ws_bytes=m.value) == L.BML_E_INVALID


def test_python_refusals(L):
    """CPU tensors are refused by name before the library is reached."""
    import bml_b200
    i, x = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, 64)
    with pytest.raises(ValueError, match="q must"):
        bml_b200.chunk_attention(x, x, x, i, i, i)
    with pytest.raises(ValueError, match="target must"):
        bml_b200.verify_drafts(x, None, i, i, i, x, x)
    with pytest.raises(ValueError, match="k_pool"):
        bml_b200.page_fork(x, x, i, i, i, i, i, i, i, i)
    with pytest.raises(ValueError, match="lens"):
        bml_b200.page_free(i, i, i, i, 16, i, i, i)
    with pytest.raises(ValueError, match="k_pool"):
        bml_b200.page_compact(x, x, i, i, i)


def test_refused_updates():
    import bml_b200
    ok = bml_b200.PageUpdate(status=torch.tensor([0, 0]))
    ok.check()
    bml_b200.PageUpdate().check()
    with pytest.raises(bml_b200.OutOfPages, match=r"\[1\]"):
        bml_b200.PageUpdate(status=torch.tensor([0, 1])).check()
    with pytest.raises(bml_b200.PageRefused, match=r"status \[8\]") as e:
        bml_b200.PageUpdate(status=torch.tensor([8, 0])).check()
    assert not isinstance(e.value, bml_b200.OutOfPages)
