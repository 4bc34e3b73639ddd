"""GPU tests of tree_attention's bounded waits: copies that never come end the
launch by themselves after a short limit and leave NaN, and the next call is
right (bml_diag_attn_tree, include/bml_diag.h)."""
import ctypes as C

import pytest
import torch

from test_paged_gpu import Paged, chain, check
from test_paged_masked_gpu import widen

pytestmark = pytest.mark.gpu

CODE = {"f32": 0, "f16": 1, "bf16": 2}


def stalled(c, qt, ct, flags, wait_ns=20_000_000):
    """The call with its own scratch, full of numbers that look like results."""
    import bml_b200
    import bml_b200._lib as L
    n, page, kv, d = c.k.shape
    out = torch.full_like(c.q, 7.0)
    ws = torch.full((bml_b200.tree_workspace_size(d) // 4,), 0.5, device="cuda")
    a = [t.data_ptr() for t in (c.q, c.k, c.v, c.table, c.kv_lens, c.start, out, ws)]
    st = L.lib().bml_diag_attn_tree(a[0], CODE[qt], c.q.shape[0], c.q.shape[1], kv, d, a[1], a[2], CODE[ct], n, page, a[3],
                                    c.table.shape[1], a[4], a[5], len(c.lens), None, 0, -1.0, a[6], a[7], ws.numel() * 4,
                                    wait_ns, flags, C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert st == 0, L.last_error()
    torch.cuda.synchronize()
    return out


# tree_umma (both chains, one row tile, two), tree_umma32, tree_few; 200 requests: a
# CTA has about ten segments, more than its copies run ahead
@pytest.mark.parametrize("qt,ct,nodes,d", [("bf16", "bf16", 20, 128), ("bf16", "bf16", 50, 128), ("f16", "f16", 20, 64),
                                           ("f32", "f32", 20, 128), ("f32", "f32", 20, 64), ("bf16", "bf16", 1, 128),
                                           ("f32", "f16", 1, 64)])
def test_stalled_copies_leave_nan(cuda, qt, ct, nodes, d):
    import bml_b200
    import bml_b200._lib as L
    lens = [(37 * i) % 300 for i in range(200)]
    c = Paged(lens, [nodes] * 200, 16, 4, d, 16, qt, ct, seed=70)
    widen(c, 16, 4096)
    out = stalled(c, qt, ct, L.BML_DIAG_STALL)
    assert torch.isnan(out).all()
    out = stalled(c, qt, ct, 0)
    assert torch.equal(out, bml_b200.tree_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.start))
    check(c, out, [chain(nodes, p) for p in lens], qt, only=[0, 1, 77, 199])
