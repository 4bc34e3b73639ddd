"""The paged KV cache and the attention of drafted tokens over it
(include/bml_attn.h, "Paged KV cache and drafted tokens").

The reference keeps one flat buffer per layer (crates/compiler/src/
kv_cache.rs:25-181 in SugarFreeDoNoSo/bml) and decodes one token of one
request at a time (gguf_compiler.rs:946-1050).  Here a request's positions
live in pages of a pool, its block table, length and page count stay on the
GPU, and one pass attends for a whole tree of drafted tokens; T = 1 is plain
decode.  A step is

  page_plan       pages, slots, positions, ancestor masks   (once a step)
  paged_append    RoPE of q and k, K and V rows stored      (every layer)
  tree_attention  attention of the new tokens               (every layer);
  chunk_attention in its place where prompts come in chunks
  verify_drafts   the path that the target's probabilities keep, and the next
                  token                                     (once a step)
  paged_commit    the accepted path moved to the front      (once a step)

and between steps page_fork lets requests share another's pages, page_free
returns pages of requests that end, page_compact packs the pool.

None of the calls waits for the GPU, and all can be captured in a CUDA
graph.  Tensors of a call live on one device, which need not be the current
one; `stream` defaults to that device's current stream.
"""
from __future__ import annotations

import ctypes as C
import warnings

import torch

from . import _lib as L
from .attention import _need, dtype_code
from .batching import MAX_PENDING_REQUESTS, AtCapacity

MAX_NODES = 256  # drafted tokens of one request in tree_attention
PLAN_NO_PAGES, PLAN_BAD, PLAN_NO_ROOM = 1, 2, 4  # status values of a plan


PAGE_SHARED = 8  # status value of a page_free


class PageRefused(RuntimeError):
    """A call that refused a request (its status says why)."""


class OutOfPages(PageRefused):
    """A plan or a fork that refused a request (its status says why)."""


# A call costs the host several microseconds and the GPU often less, so the
# usual ones (plain tensors, the current device and stream) are made by a module
# in C++ (_load); what it leaves alone is checked and called below, with one
# test per tensor on the way that is right (_bad says what is wrong on the
# other), raw stream handles and addresses, few allocations.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _bad(t, name: str, dtype=None, ndim=None, shape=None, device=None):
    """Raises the error that says what is wrong with an argument."""
    _need(t, name, dtype, ndim)
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    raise ValueError(f"{name} is not a valid argument")


def _ints(t, name: str, device, shape=None, ndim: int = 1, dtype=torch.int32) -> int:
    """The address of a contiguous integer tensor on `device`."""
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or not t.is_contiguous()
            or (t.shape != shape if shape is not None else t.dim() != ndim)):
        _bad(t, name, dtype, None if shape is not None else ndim, shape, device)
    return t.data_ptr()


def _data(t, name: str, ndim: int, dtype=None, device=None) -> int:
    """The address of a contiguous CUDA tensor."""
    if (not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != ndim or not t.is_contiguous()
            or (dtype is not None and t.dtype is not dtype) or (device is not None and t.device != device)):
        _bad(t, name, dtype, ndim, None, device)
    return t.data_ptr()


def _enter(device: torch.device, stream):
    """Makes the device current, and the stream where one is given, so that
    the buffers a call allocates belong to the stream that uses them.  None in
    the usual case, where both are; else a context that has been entered."""
    if stream is None:
        if device.index == _current_device():
            return None
        ctx = torch.cuda.device(device)
    else:
        if stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
        ctx = torch.cuda.stream(stream)
    ctx.__enter__()
    return ctx


_fast = None  # csrc/torch_calls.cpp: the usual calls without Python's share of the time


class _Wrappers:
    """In that module's place: leaves every call to the wrappers below."""

    @staticmethod
    def plan(*args):
        return None

    append = tree = commit = plan
    chunk = verify = fork = free = compact = plan


def _load():
    """Loads that module and gives it the library's entry points.  One that is
    missing or was built for another torch is not used: the calls are the same
    through ctypes, 4 to 15 us slower on the host."""
    global _fast
    lib = L.lib()
    try:
        from . import _torch_calls
        found = _torch_calls.built_for
    except (ImportError, AttributeError) as e:  # none, symbols that this torch lacks, or an older build
        found = str(e)
    if found != torch.__version__:
        warnings.warn(f"bml_b200/_torch_calls.so is not for torch {torch.__version__} ({found}): paged calls go through ctypes; "
                      "build it with `python -m bml_b200.build`", RuntimeWarning, stacklevel=3)
        _fast = _Wrappers
        return _fast
    _torch_calls.set_calls(*(C.cast(getattr(lib, f), C.c_void_p).value for f in (
        "bml_paged_plan", "bml_paged_append", "bml_attn_tree_sized", "bml_paged_commit", "bml_attn_tree_workspace_size",
        "bml_attn_chunk", "bml_attn_chunk_workspace_size", "bml_verify_drafts", "bml_page_fork", "bml_page_free",
        "bml_page_compact")))
    _fast = _torch_calls
    return _fast


_fns: dict = {}


def _call(fn: str, *args) -> None:
    f = _fns.get(fn)
    if f is None:
        f = _fns[fn] = getattr(L.lib(), fn)
    status = f(*args)
    if status:
        L.check(status, fn)


class PagePlan:
    """One step's plan; all tensors on the device (see bml_paged_plan).

    node_start int32 [n + 1], kv_lens, owned, status int32 [n], free_used
    int32 [1], slots int64 [n_tokens], positions int32 [n_tokens], mask int64
    [n_tokens, n_words] (None without parents)."""

    __slots__ = ("node_start", "kv_lens", "owned", "free_used", "status", "positions", "slots", "mask")

    def check(self) -> None:
        """Raises OutOfPages if a request was refused.  Waits for the GPU."""
        bad = self.status.nonzero().flatten().tolist()
        if bad:
            raise OutOfPages(f"requests {bad} refused, status {self.status[bad].tolist()}")


def page_plan(lens: torch.Tensor, n_new: torch.Tensor, owned: torch.Tensor, block_table: torch.Tensor,
              free_pages: torch.Tensor, free_used: torch.Tensor, page_size: int, n_tokens: int,
              parents: torch.Tensor | None = None, n_words: int = 1, stream=None) -> PagePlan:
    """Plans one step of n requests: pages for n_new[i] new tokens behind
    lens[i] positions, taken from free_pages[free_used:] in request order and
    written into block_table [n, max_pages]; the tokens' slots and positions,
    and with `parents` [n_tokens] their ancestor masks.  lens, n_new, owned
    [n], free_pages, free_used [1] are int32; n_tokens is the row count of
    the step's token arrays, at least the sum of n_new.  lens, owned and
    free_used are not changed: the plan carries their next values."""
    if stream is None:
        r = (_fast or _load()).plan(lens, n_new, owned, block_table, free_pages, free_used, page_size, n_tokens, parents,
                                    n_words)
        if r is not None:
            p = PagePlan()
            p.node_start, p.kv_lens, p.owned, p.free_used, p.status, p.positions, p.slots, p.mask = r
            return p
    dev = lens.device if isinstance(lens, torch.Tensor) else None
    if dev is None or dev.type != "cuda":
        _bad(lens, "lens", torch.int32, 1)
    a_lens = _ints(lens, "lens", dev)
    one = lens.shape
    n = one[0]
    a_new, a_owned = _ints(n_new, "n_new", dev, one), _ints(owned, "owned", dev, one)
    a_table = _ints(block_table, "block_table", dev, ndim=2)
    rows, max_pages = block_table.shape
    if rows != n:
        raise ValueError(f"block_table must be [{n}, max_pages], got {tuple(block_table.shape)}")
    a_free, a_used = _ints(free_pages, "free_pages", dev), _ints(free_used, "free_used", dev, (1,))
    if not (0 <= n_tokens < 1 << 31 and 0 <= page_size < 1 << 31):  # ctypes would cut them to 32 bits
        raise ValueError(f"n_tokens {n_tokens} and page_size {page_size} must be 0 to 2^31 - 1")
    a_parents = None
    if parents is not None:
        a_parents = _ints(parents, "parents", dev, (n_tokens,))
        if not 1 <= n_words <= MAX_NODES // 64:
            raise ValueError(f"n_words must be 1 to {MAX_NODES // 64}, got {n_words}")
    p = PagePlan()
    ctx = _enter(dev, stream)
    try:
        p.slots = torch.empty(n_tokens, dtype=torch.int64, device=dev)
        p.mask = a_mask = None
        if parents is not None:
            p.mask = torch.empty((n_tokens, n_words), dtype=torch.int64, device=dev)
            a_mask = p.mask.data_ptr()
        small = torch.empty(4 * n + 2 + n_tokens, dtype=torch.int32, device=dev)  # the int32 arrays
        a = small.data_ptr()
        b = a + 4 * n_tokens
        _call("bml_paged_plan", a_lens, a_new, a_owned, n, a_free, free_pages.shape[0], a_used, page_size, max_pages,
              a_table, a_parents, n_tokens, n_words, b, b + 4 * (n + 1), b + 4 * (2 * n + 1), b + 4 * (4 * n + 1),
              p.slots.data_ptr(), a, a_mask, b + 4 * (3 * n + 1), _raw_stream(dev.index))
    finally:
        if ctx is not None:
            ctx.__exit__(None, None, None)
    p.positions, p.node_start, p.kv_lens, p.owned, p.status, p.free_used = torch.unsafe_split_with_sizes(
        small, (n_tokens, n + 1, n, n, n, 1))
    return p


def _pools(k_pool, v_pool, ndim: int, device=None):
    """The pools' addresses and shape."""
    a = _data(k_pool, "k_pool", ndim, None, device)
    b = _data(v_pool, "v_pool", ndim, k_pool.dtype, k_pool.device)
    shape = k_pool.shape
    if shape != v_pool.shape:
        raise ValueError(f"k_pool {tuple(shape)} and v_pool {tuple(v_pool.shape)} do not match")
    return a, b, shape


def paged_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
                 positions: torch.Tensor | None, k_pool: torch.Tensor, v_pool: torch.Tensor,
                 q_out: torch.Tensor | None = None, theta: float = 10000.0, stream=None) -> torch.Tensor | None:
    """RoPE and store of one layer's new tokens: q [n, n_heads, d] turned by
    positions [n] int32 (in place, or into q_out), k turned and v as is
    ([n, n_kv, d]) into row slots[t] (int64) of the pools
    [n_pages, page_size, n_kv, d].  q, k, v in one type (f32, f16, bf16), the
    pools in any.  positions None: no rotation; q None: no queries.  A token
    whose slot is -1 (or outside the pool) is skipped.  Returns the turned q."""
    if stream is None:
        r = (_fast or _load()).append(q, k, v, slots, positions, k_pool, v_pool, q_out, theta)
        if r is not None:
            return None if r is True else r
    a_k = _data(k, "k", 3)
    dev, dtype = k.device, k.dtype
    a_v = _data(v, "v", 3, dtype, dev)
    shape = k.shape
    n, n_kv, d = shape
    if shape != v.shape:
        raise ValueError(f"k {tuple(shape)} and v {tuple(v.shape)} do not match")
    a_kp, a_vp, pool = _pools(k_pool, v_pool, 4, dev)
    if pool[2] != n_kv or pool[3] != d:
        raise ValueError(f"pool rows {tuple(pool[2:])} do not match k {tuple(shape)}")
    a_slots = _ints(slots, "slots", dev, (n,), dtype=torch.int64)
    a_pos = None if positions is None else _ints(positions, "positions", dev, (n,))
    n_heads, a_q, a_out = 0, None, None
    if q is not None:
        a_q = a_out = _data(q, "q", 3, dtype, dev)
        q_shape = q.shape
        n_heads = q_shape[1]
        if q_shape[0] != n or q_shape[2] != d:
            raise ValueError(f"q {tuple(q_shape)} does not match k {tuple(shape)}")
        if q_out is None:
            q_out = q
        else:
            a_out = _data(q_out, "q_out", 3, dtype, dev)
            if q_out.shape != q_shape:
                raise ValueError(f"q_out {tuple(q_out.shape)} does not match q {tuple(q_shape)}")
    elif q_out is not None:
        raise ValueError("q_out without q")
    ctx = _enter(dev, stream)
    try:
        _call("bml_paged_append", a_q, a_k, a_v, dtype_code(dtype), a_slots, a_pos, n, n_heads, n_kv, d, theta, a_out,
              a_kp, a_vp, dtype_code(k_pool.dtype), pool[0] * pool[1], _raw_stream(dev.index))
    finally:
        if ctx is not None:
            ctx.__exit__(None, None, None)
    return q_out


_ws_bytes: dict = {}


def tree_workspace_size(head_dim: int, device=None) -> int:
    """Scratch bytes of tree_attention on a device (whatever the batch)."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index or 0
    key = (dev, head_dim)
    if key not in _ws_bytes:
        size = C.c_size_t()
        L.call("bml_attn_tree_workspace_size", head_dim, dev, C.byref(size))
        _ws_bytes[key] = size.value
    return _ws_bytes[key]


def tree_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                   kv_lens: torch.Tensor, node_start: torch.Tensor, mask: torch.Tensor | None = None,
                   scale: float = -1.0, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                   stream=None, n_live: int = 0, max_new: int = 0) -> torch.Tensor:
    """Attention of every request's new tokens over its pages.  q
    [n_tokens, n_heads, d] holds request i's T tokens in rows
    node_start[i]..node_start[i+1]; a token attends over the request's first
    kv_lens[i] - T positions and over the new tokens that its mask row
    (int64 [n_tokens, 1 to 4], bit j: the request's j-th new token) names;
    without a mask, over itself and those before it (T = 1: plain decode).
    q is f32, or of the pools' 16-bit type; the result has q's type.  At most
    256 new tokens a request (64 a mask word).  Rows that see nothing, and
    those of requests that page_plan refused or that have more new tokens, are
    zero; rows behind the last request's are not written (in a result that the
    call allocates they hold anything).  scale < 0 selects 1/sqrt(d).

    workspace: an uint8 tensor of tree_workspace_size bytes for calls that
    must not allocate; calls that share one must not overlap.  By default
    scratch comes from torch's allocator, on the call's stream.

    n_live, max_new: how many requests have new tokens, and the most of one,
    where the host knows it (0: not).  The kernel is chosen by them, else by the
    average over all requests; results are right whatever they say."""
    if stream is None and out is None and workspace is None:
        r = (_fast or _load()).tree(q, k_pool, v_pool, block_table, kv_lens, node_start, mask, scale,
                                    n_live, max_new)
        if r is not None:
            return r
    a_q = _data(q, "q", 3)
    shape, dev, dtype = q.shape, q.device, q.dtype
    n_tokens, n_heads, d = shape
    a_k, a_v, pool = _pools(k_pool, v_pool, 4, dev)
    n_pages, page_size, n_kv, pd = pool
    if pd != d:
        raise ValueError(f"q {tuple(shape)} does not match the pools {tuple(pool)}")
    a_len = _ints(kv_lens, "kv_lens", dev)
    n = kv_lens.shape[0]
    a_start = _ints(node_start, "node_start", dev, (n + 1,))
    a_table = _ints(block_table, "block_table", dev, ndim=2)
    rows, max_pages = block_table.shape
    if rows != n:
        raise ValueError(f"block_table must be [{n}, max_pages], got {tuple(block_table.shape)}")
    a_mask, n_words = None, 0
    if mask is not None:
        a_mask = _ints(mask, "mask", dev, ndim=2, dtype=torch.int64)
        rows, n_words = mask.shape
        if rows != n_tokens or not 1 <= n_words <= MAX_NODES // 64:
            raise ValueError(f"mask must be [{n_tokens}, 1 to {MAX_NODES // 64}], got {tuple(mask.shape)}")
    if not (0 <= n_live <= 0x7fffffff and 0 <= max_new <= 0x7fffffff):
        raise ValueError("n_live and max_new must not be negative")
    ctx = _enter(dev, stream)
    try:
        if out is None:
            out = torch.empty_like(q)
        elif _data(out, "out", 3, dtype, dev) and out.shape != shape:
            raise ValueError(f"out {tuple(out.shape)} does not match q {tuple(shape)}")
        if workspace is None:
            need = _ws_bytes.get((dev.index, d)) or tree_workspace_size(d, dev)
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        else:
            _ints(workspace, "workspace", dev, dtype=torch.uint8)
        _call("bml_attn_tree_sized", a_q, dtype_code(dtype), n_tokens, n_heads, n_kv, d, a_k, a_v, dtype_code(k_pool.dtype),
              n_pages, page_size, a_table, max_pages, a_len, a_start, n, a_mask, n_words, scale, out.data_ptr(),
              workspace.data_ptr(), workspace.shape[0], n_live, max_new, _raw_stream(dev.index))
    finally:
        if ctx is not None:
            ctx.__exit__(None, None, None)
    return out


def paged_commit(k_pools: torch.Tensor, v_pools: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                 kv_lens: torch.Tensor, node_start: torch.Tensor, path: torch.Tensor, n_accept: torch.Tensor,
                 stream=None) -> torch.Tensor:
    """Moves the accepted path of every request's draft behind its committed
    positions, in the pools [n_layers, n_pages, page_size, n_kv, d] of all
    layers: row lens[i] + path[i, k] to lens[i] + k for k < n_accept[i].
    path [n, max_path] int32 holds strictly increasing node indices; an entry
    that is not ends the path.  Returns the new lengths int32 [n]; a request
    that page_plan refused keeps its own."""
    if stream is None:
        r = (_fast or _load()).commit(k_pools, v_pools, block_table, lens, kv_lens, node_start, path, n_accept)
        if r is not None:
            return r
    a_k, a_v, pool = _pools(k_pools, v_pools, 5)
    layers, n_pages, page_size, n_kv, d = pool
    dev = k_pools.device
    a_lens = _ints(lens, "lens", dev)
    one = lens.shape
    n = one[0]
    a_len, a_start = _ints(kv_lens, "kv_lens", dev, one), _ints(node_start, "node_start", dev, (n + 1,))
    a_accept, a_table = _ints(n_accept, "n_accept", dev, one), _ints(block_table, "block_table", dev, ndim=2)
    a_path = _ints(path, "path", dev, ndim=2)
    rows, max_pages = block_table.shape
    path_rows, max_path = path.shape
    if rows != n:
        raise ValueError(f"block_table must be [{n}, max_pages], got {tuple(block_table.shape)}")
    if path_rows != n:
        raise ValueError(f"path must be [{n}, max_path], got {tuple(path.shape)}")
    ctx = _enter(dev, stream)
    try:
        new = torch.empty_like(lens)
        _call("bml_paged_commit", a_k, a_v, layers, n_pages, page_size, n_kv, d, dtype_code(k_pools.dtype), a_table,
              max_pages, a_lens, a_len, a_start, n, a_path, max_path, a_accept, new.data_ptr(),
              _raw_stream(dev.index))
    finally:
        if ctx is not None:
            ctx.__exit__(None, None, None)
    return new


def chunk_workspace_size(head_dim: int, n_tokens: int, n_requests: int, device=None) -> int:
    """Scratch bytes of chunk_attention for a batch of that size."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index or 0
    size = C.c_size_t()
    L.call("bml_attn_chunk_workspace_size", head_dim, n_tokens, n_requests, dev, C.byref(size))
    return size.value


def chunk_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, node_start: torch.Tensor, scale: float = -1.0,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None, n_live: int = 0,
                    max_new: int = 0) -> torch.Tensor:
    """Attention of chunks of new tokens over pages: tree_attention without a
    mask, for any number of new tokens a request -- a prompt or a part of one,
    beside requests that decode one token.  The j-th of request i's T new tokens
    (row node_start[i] + j of q) attends over positions 0 to kv_lens[i] - T + j.
    Types, results, refused requests and rows behind the last request's are
    tree_attention's, and so are n_live and max_new.  workspace: an uint8 tensor of
    chunk_workspace_size bytes (up to 158 MB from 1024 tokens on) for calls that must
    not allocate; calls that share one must not overlap.  For batches of single
    tokens tree_attention is the faster call (include/bml_attn.h has figures)."""
    if stream is None and out is None and workspace is None:
        r = (_fast or _load()).chunk(q, k_pool, v_pool, block_table, kv_lens, node_start, scale, n_live, max_new)
        if r is not None:
            return r
    a_q = _data(q, "q", 3)
    shape, dev, dtype = q.shape, q.device, q.dtype
    n_tokens, n_heads, d = shape
    a_k, a_v, pool = _pools(k_pool, v_pool, 4, dev)
    n_pages, page_size, n_kv, pd = pool
    if pd != d:
        raise ValueError(f"q {tuple(shape)} does not match the pools {tuple(pool)}")
    a_len = _ints(kv_lens, "kv_lens", dev)
    n = kv_lens.shape[0]
    a_start = _ints(node_start, "node_start", dev, (n + 1,))
    a_table = _ints(block_table, "block_table", dev, ndim=2)
    rows, max_pages = block_table.shape
    if rows != n:
        raise ValueError(f"block_table must be [{n}, max_pages], got {tuple(block_table.shape)}")
    if not (0 <= n_live <= 0x7fffffff and 0 <= max_new <= 0x7fffffff):
        raise ValueError("n_live and max_new must not be negative")
    ctx = _enter(dev, stream)
    try:
        if out is None:
            out = torch.empty_like(q)
        elif _data(out, "out", 3, dtype, dev) and out.shape != shape:
            raise ValueError(f"out {tuple(out.shape)} does not match q {tuple(shape)}")
        if workspace is None:
            workspace = torch.empty(chunk_workspace_size(d, n_tokens, n, dev), dtype=torch.uint8, device=dev)
        else:
            _ints(workspace, "workspace", dev, dtype=torch.uint8)
        _call("bml_attn_chunk", a_q, dtype_code(dtype), n_tokens, n_heads, n_kv, d, a_k, a_v, dtype_code(k_pool.dtype),
              n_pages, page_size, a_table, max_pages, a_len, a_start, n, scale, out.data_ptr(), workspace.data_ptr(),
              workspace.shape[0], n_live, max_new, _raw_stream(dev.index))
    finally:
        if ctx is not None:
            ctx.__exit__(None, None, None)
    return out


def verify_drafts(target: torch.Tensor, draft: torch.Tensor | None, tokens: torch.Tensor, parents: torch.Tensor,
                  node_start: torch.Tensor, u: torch.Tensor, u_next: torch.Tensor, max_path: int = MAX_NODES,
                  stream=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which path of each request's draft the target model keeps, and the token
    that follows it, so that tokens are distributed as the target's.  Request
    i's nodes are rows node_start[i]..node_start[i+1]; node 0 is its pending token
    and always kept, a node whose parent is an earlier node is a drafted child of
    it, any other is never kept.  target [n_tokens, vocab]: the target's
    probabilities behind each node; draft: those (of the same type) that each
    node's children were drawn from, independently, or None for tokens that were
    picked; tokens, parents int32 [n_tokens]; u [n_tokens] and u_next [n] f32:
    random numbers in [0, 1).  Rows are distributions: where a draft row is none (it
    sums to more than twice the target's) and nothing is left to draw from, the
    next token is vocab - 1, which then means nothing.

    Returns path int32 [n, max_path] (-1 behind its end) and n_accept [n], as
    paged_commit takes them, and the next tokens int32 [n].  At a kept node its
    children are tried in node order: x is kept with probability min(1, r(x) /
    q(x)), r the target's probabilities at first and norm(max(r - q, 0)) after
    each rejection; if none is, the next token is drawn from r.  A path of
    max_path nodes ends there.  A request without nodes, or with more than 256,
    has n_accept 0 and next -1; one that page_plan refused is walked like any other
    (look at its status).  include/bml_attn.h has the formulas."""
    if stream is None:
        r = (_fast or _load()).verify(target, draft, tokens, parents, node_start, u, u_next, max_path)
        if r is not None:
            return r
    a_t = _data(target, "target", 2)
    dev, dtype = target.device, target.dtype
    rows, vocab = target.shape
    a_d = None
    if draft is not None:
        a_d = _data(draft, "draft", 2, dtype, dev)
        if draft.shape != target.shape:
            raise ValueError(f"draft {tuple(draft.shape)} does not match target {tuple(target.shape)}")
    a_tok, a_par = _ints(tokens, "tokens", dev, (rows,)), _ints(parents, "parents", dev, (rows,))
    a_start = _ints(node_start, "node_start", dev)
    n = node_start.shape[0] - 1
    a_u, a_next = _ints(u, "u", dev, (rows,), dtype=torch.float32), _ints(u_next, "u_next", dev, (n,), dtype=torch.float32)
    if not 1 <= max_path < 1 << 31:
        raise ValueError(f"max_path must be 1 to 2^31 - 1, got {max_path}")
    ctx = _enter(dev, stream)
    try:
        path = torch.empty((n, max_path), dtype=torch.int32, device=dev)
        count, token = torch.empty((2, n), dtype=torch.int32, device=dev).unbind()
        _call("bml_verify_drafts", a_t, a_d, dtype_code(dtype), vocab, a_tok, a_par, rows, a_start, n, a_u, a_next,
              max_path, path.data_ptr(), count.data_ptr(), token.data_ptr(), _raw_stream(dev.index))
    finally:
        if ctx is not None:
            ctx.__exit__(None, None, None)
    return path, count, token


class PageUpdate:
    """What page_fork, page_free and page_compact make of the pages' state: the
    arrays that the call replaces (None: it leaves that one as it is).

    lens, owned int32 [n], shared int32 [n_pages], free_pages int32 [n_free],
    free_used int32 [1], block_table int32 [n, max_pages], status int32."""

    __slots__ = ("lens", "owned", "shared", "free_pages", "free_used", "block_table", "status")

    def __init__(self, lens=None, owned=None, shared=None, free_pages=None, free_used=None, block_table=None, status=None):
        self.lens, self.owned, self.shared, self.free_pages = lens, owned, shared, free_pages
        self.free_used, self.block_table, self.status = free_used, block_table, status

    def check(self) -> None:
        """Raises OutOfPages or PageRefused if something was refused.  Waits for the GPU."""
        bad = [] if self.status is None else self.status.nonzero().flatten().tolist()
        if bad:
            status = self.status[bad].tolist()
            raise (OutOfPages if PLAN_NO_PAGES in status else PageRefused)(f"entries {bad} refused, status {status}")


def page_fork(k_pools: torch.Tensor, v_pools: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, lens: torch.Tensor,
              owned: torch.Tensor, block_table: torch.Tensor, shared: torch.Tensor, free_pages: torch.Tensor,
              free_used: torch.Tensor, stream=None) -> PageUpdate:
    """Lets row dst[j] of the tables continue the positions of row src[j], in the
    pools [n_layers, n_pages, page_size, n_kv, d] of all layers: full pages are
    shared (shared [n_pages] counts a page's holders beyond the first), the rows of
    a part-filled one are copied to a page of the free list.  src, dst [m], lens,
    owned [n], block_table [n, max_pages] (rows dst written), free_pages, free_used
    [1]: int32, as page_plan takes them.  dst must be idle rows.  Returns the next
    lens, owned, shared and free_used, and a status per fork."""
    if stream is None:
        r = (_fast or _load()).fork(k_pools, v_pools, src, dst, lens, owned, block_table, shared, free_pages, free_used)
        if r is not None:
            return PageUpdate(r[0], r[1], r[2], None, r[3], None, r[4])
    a_k, a_v, pool = _pools(k_pools, v_pools, 5)
    layers, n_pages, page_size, n_kv, d = pool
    dev = k_pools.device
    a_src = _ints(src, "src", dev)
    m = src.shape[0]
    a_dst = _ints(dst, "dst", dev, (m,))
    a_lens = _ints(lens, "lens", dev)
    n = lens.shape[0]
    a_owned, a_table = _ints(owned, "owned", dev, (n,)), _ints(block_table, "block_table", dev, ndim=2)
    if block_table.shape[0] != n:
        raise ValueError(f"block_table must be [{n}, max_pages], got {tuple(block_table.shape)}")
    a_shared = _ints(shared, "shared", dev, (n_pages,))
    a_free, a_used = _ints(free_pages, "free_pages", dev), _ints(free_used, "free_used", dev, (1,))
    ctx = _enter(dev, stream)
    try:
        buf = torch.empty(2 * n + n_pages + 1 + m, dtype=torch.int32, device=dev)
        out = torch.unsafe_split_with_sizes(buf, (n, n, n_pages, 1, m))
        _call("bml_page_fork", a_k, a_v, layers, n_pages, page_size, n_kv, d, dtype_code(k_pools.dtype), a_src, a_dst, m,
              a_lens, a_owned, n, a_table, block_table.shape[1], a_shared, a_free, free_pages.shape[0], a_used,
              *(x.data_ptr() for x in out), _raw_stream(dev.index))
    finally:
        if ctx is not None:
            ctx.__exit__(None, None, None)
    return PageUpdate(out[0], out[1], out[2], None, out[3], None, out[4])


def page_free(keep: torch.Tensor, lens: torch.Tensor, owned: torch.Tensor, block_table: torch.Tensor, page_size: int,
              shared: torch.Tensor, free_pages: torch.Tensor, free_used: torch.Tensor, stream=None) -> PageUpdate:
    """Ends or rolls back requests: request i keeps min(lens[i], keep[i])
    positions (negative: everything) and the pages that hold them; pages that
    all their holders have released return to the free list, whose taken part is
    parted into pages still held and freed ones.  Refused (status 8) where keep ends
    inside a page that others hold.  keep, lens, owned [n], block_table [n,
    max_pages], shared [n_pages], free_pages, free_used [1] are int32.  Returns the
    next lens, owned, shared, free_pages and free_used, and a status per request."""
    if stream is None:
        r = (_fast or _load()).free(keep, lens, owned, block_table, page_size, shared, free_pages, free_used)
        if r is not None:
            return PageUpdate(r[0], r[1], r[2], r[3], r[4], None, r[5])
    dev = lens.device if isinstance(lens, torch.Tensor) else None
    if dev is None or dev.type != "cuda":
        _bad(lens, "lens", torch.int32, 1)
    a_lens = _ints(lens, "lens", dev)
    n = lens.shape[0]
    a_keep, a_owned = _ints(keep, "keep", dev, (n,)), _ints(owned, "owned", dev, (n,))
    a_table = _ints(block_table, "block_table", dev, ndim=2)
    if block_table.shape[0] != n:
        raise ValueError(f"block_table must be [{n}, max_pages], got {tuple(block_table.shape)}")
    a_shared, a_free = _ints(shared, "shared", dev), _ints(free_pages, "free_pages", dev)
    a_used = _ints(free_used, "free_used", dev, (1,))
    n_pages, n_free = shared.shape[0], free_pages.shape[0]
    if not 0 <= page_size < 1 << 31:  # ctypes would cut it to 32 bits
        raise ValueError(f"page_size {page_size} must be 0 to 2^31 - 1")
    ctx = _enter(dev, stream)
    try:
        work = 1024 + (n_free + 31) // 32
        buf = torch.empty(3 * n + n_pages + n_free + 1 + work, dtype=torch.int32, device=dev)
        out = torch.unsafe_split_with_sizes(buf, (n, n, n_pages, n_free, 1, n, work))
        _call("bml_page_free", a_keep, a_lens, a_owned, n, a_table, block_table.shape[1], page_size, a_shared, n_pages,
              a_free, n_free, a_used, *(x.data_ptr() for x in out), 4 * work, _raw_stream(dev.index))
    finally:
        if ctx is not None:
            ctx.__exit__(None, None, None)
    return PageUpdate(out[0], out[1], out[2], out[3], out[4], None, out[5])


def page_compact(k_pools: torch.Tensor, v_pools: torch.Tensor, owned: torch.Tensor, block_table: torch.Tensor,
                 shared: torch.Tensor, stream=None) -> PageUpdate:
    """Packs the pools [n_layers, n_pages, page_size, n_kv, d]: the H held pages (the
    first owned[i] entries of each row of block_table) come to lie at 0 to H - 1.
    Those behind move, in ascending order, into the pages below H that nobody holds.
    owned [n], block_table [n, max_pages], shared [n_pages] are int32.  Returns the
    next block_table, shared, free_pages (0, 1, 2, ...) and free_used (H)."""
    if stream is None:
        r = (_fast or _load()).compact(k_pools, v_pools, owned, block_table, shared)
        if r is not None:
            return PageUpdate(None, None, r[1], r[2], r[3], r[0])
    a_k, a_v, pool = _pools(k_pools, v_pools, 5)
    layers, n_pages, page_size, n_kv, d = pool
    dev = k_pools.device
    a_owned, a_table = _ints(owned, "owned", dev), _ints(block_table, "block_table", dev, ndim=2)
    n, max_pages = owned.shape[0], block_table.shape[1]
    if block_table.shape[0] != n:
        raise ValueError(f"block_table must be [{n}, max_pages], got {tuple(block_table.shape)}")
    a_shared = _ints(shared, "shared", dev, (n_pages,))
    ctx = _enter(dev, stream)
    try:
        table, work = torch.empty_like(block_table), torch.empty(3 * n_pages + 1, dtype=torch.int32, device=dev)
        out = torch.unsafe_split_with_sizes(torch.empty(2 * n_pages + 1, dtype=torch.int32, device=dev),
                                            (n_pages, n_pages, 1))
        _call("bml_page_compact", a_k, a_v, layers, n_pages, page_size, n_kv, d, dtype_code(k_pools.dtype), a_owned, n,
              a_table, max_pages, a_shared, table.data_ptr(), *(x.data_ptr() for x in out), work.data_ptr(),
              4 * work.shape[0], _raw_stream(dev.index))
    finally:
        if ctx is not None:
            ctx.__exit__(None, None, None)
    return PageUpdate(None, None, out[0], out[1], out[2], table)


def _on(device, values) -> torch.Tensor:
    """int32 values of the host on the device, without waiting for the GPU as a copy
    from pageable memory does.  Torch's allocator keeps the pinned block until the
    copy has been made; only memory that it has to pin anew waits.  A graph would
    replay the copy from a block that holds something else by then."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a PagedBatcher's host state cannot be captured: plan, commit and remove outside the graph")
    return torch.tensor(values, dtype=torch.int32, pin_memory=True).to(device, non_blocking=True)


class PagedBatcher:
    """DecodeBatcher over a paged cache, with drafts: requests join and leave
    between steps, a step brings each request any number of new tokens -- one
    to decode, a chain, or a tree of drafted tokens -- and commit() keeps the
    accepted ones.  Prompts may come in chunks of any length beside them.

    Per step: ``begin(new)`` plans it; for every layer ``step(layer, q, k, v)``
    stores the tokens and returns their attention; ``commit(paths)`` ends it, or
    ``verify(...)``, which finds the paths on the GPU.  Token rows are the
    requests' tokens in the order of ``active``.  Between steps ``fork`` lets
    requests continue another's positions, ``truncate`` rolls one back, and
    ``compact`` packs the pool."""

    def __init__(self, n_layers: int, n_heads: int, n_kv_heads: int, head_dim: int, n_pages: int,
                 page_size: int = 64, max_positions: int = 8192, dtype: torch.dtype = torch.bfloat16, device=None,
                 rope: bool = True, theta: float = 10000.0, max_requests: int = MAX_PENDING_REQUESTS,
                 scale: float = -1.0):
        if n_heads % n_kv_heads:
            raise ValueError("n_heads must be a multiple of n_kv_heads")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim {head_dim} (supported: 64, 128)")
        dtype_code(dtype)
        self.n_layers, self.n_heads, self.n_kv, self.head_dim = n_layers, n_heads, n_kv_heads, head_dim
        self.page_size, self.rope, self.theta, self.scale = page_size, rope, float(theta), float(scale)
        self.max_requests = max_requests
        self.device = torch.device("cuda", torch.cuda.current_device() if device is None else
                                   torch.device(device).index or 0)
        shape = (n_layers, n_pages, page_size, n_kv_heads, head_dim)
        # uninitialised: attention reads no row that no append has written
        self.k = torch.empty(shape, dtype=dtype, device=self.device)
        self.v = torch.empty(shape, dtype=dtype, device=self.device)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.table = torch.full((max_requests, -(-max_positions // page_size)), -1, **i32)
        self.lens, self.owned = torch.zeros(max_requests, **i32), torch.zeros(max_requests, **i32)
        self.free, self.used = torch.arange(n_pages, **i32), torch.zeros(1, **i32)
        self.shared = torch.zeros(n_pages, **i32)  # holders of a page beyond the first
        self._rows: dict = {}    # request -> its row of the tables
        self._plan = None        # of the step that has begun,
        self._checked = True     # and whether it refused nobody, as far as the host knows
        self._new = None         # new tokens of each row (host),
        self._live = self._most = 0  # how many rows have some, the most of one
        self._parents = []       # of the step's tokens (host)

    @property
    def active(self) -> list:
        return sorted(self._rows, key=self._rows.get)

    def __len__(self) -> int:
        return len(self._rows)

    def length(self, rid) -> int:
        """Committed positions of a request.  Waits for the GPU."""
        return int(self.lens[self._rows[rid]])

    def add(self, rid, k_prompt: torch.Tensor | None = None, v_prompt: torch.Tensor | None = None) -> None:
        """Admits a request; the prompt's K/V ([n_layers, P, n_kv, d], e.g.
        from a prefill, RoPE applied) become its first P positions."""
        if self._plan is not None:
            raise RuntimeError("a step has begun: commit it first")
        if rid in self._rows:
            raise KeyError(f"request {rid!r} is already active")
        if len(self._rows) >= self.max_requests:
            raise AtCapacity(f"{len(self._rows)} requests active (max {self.max_requests})")
        if (k_prompt is None) != (v_prompt is None):
            raise ValueError("k_prompt and v_prompt come together")
        if k_prompt is not None:
            want = (self.n_layers, k_prompt.shape[1] if k_prompt.dim() == 4 else -1, self.n_kv, self.head_dim)
            if tuple(k_prompt.shape) != want or k_prompt.shape != v_prompt.shape:
                raise ValueError(f"prompt K/V {tuple(k_prompt.shape)} / {tuple(v_prompt.shape)} do not match")
        self._rows[rid] = min(set(range(self.max_requests)) - set(self._rows.values()))
        if k_prompt is None or k_prompt.shape[1] == 0:
            return
        n = k_prompt.shape[1]
        try:
            plan = self._planned({rid: n})
            plan.check()
            for layer in range(self.n_layers):
                paged_append(None, k_prompt[layer].contiguous(), v_prompt[layer].contiguous(), plan.slots, None,
                             self.k[layer], self.v[layer])
        except Exception:
            del self._rows[rid]  # and its pages stay free: owned and used are those before the plan
            raise
        self.owned, self.used, self.lens = plan.owned, plan.free_used, plan.kv_lens + self._idle(plan)

    def _idle(self, plan: PagePlan) -> torch.Tensor:
        """Lengths of the refused requests (kv_lens gives them as 0)."""
        return torch.where(plan.status != 0, self.lens, torch.zeros_like(self.lens))

    def _between_steps(self) -> None:
        if self._plan is not None:
            raise RuntimeError("a step has begun: commit it first")

    def _keep(self, rows: dict, check: bool) -> None:
        """Releases what the given rows hold behind so many positions."""
        keep = [rows.get(r, -1) for r in range(self.max_requests)]
        p = page_free(_on(self.device, keep), self.lens, self.owned, self.table,
                      self.page_size, self.shared, self.free, self.used)
        if check:
            p.check()
        self.lens, self.owned, self.shared = p.lens, p.owned, p.shared
        self.free, self.used = p.free_pages, p.free_used

    def remove(self, rid) -> None:
        """Drops a request and returns the pages that no other one shares, without
        waiting for the GPU."""
        self._between_steps()
        self._keep({self._rows[rid]: 0}, False)
        del self._rows[rid]

    def truncate(self, rid, n: int) -> None:
        """Rolls a request back to its first n positions.  PageRefused where that
        ends inside a page that it shares.  Waits for the GPU."""
        self._between_steps()
        if n < 0:
            raise ValueError(f"{n} positions")
        self._keep({self._rows[rid]: n}, True)

    def fork(self, rid, new) -> None:
        """Admits a request, or a list of them, that continues the positions of
        `rid`: its full pages are shared, a part-filled one is copied.  OutOfPages
        where the pool has no page for that; then none is admitted.  Waits for
        the GPU."""
        self._between_steps()
        new = list(new) if isinstance(new, list) else [new]  # (a tuple may be a request's name, as in add)
        row = self._rows[rid]
        if len(set(new)) < len(new) or any(r in self._rows for r in new):
            raise KeyError(f"requests {new!r}: one is already active, or named twice")
        if len(self._rows) + len(new) > self.max_requests:
            raise AtCapacity(f"{len(self._rows)} requests active (max {self.max_requests}), {len(new)} more")
        if not new:
            return
        free = sorted(set(range(self.max_requests)) - set(self._rows.values()))[:len(new)]
        p = page_fork(self.k, self.v, _on(self.device, [row] * len(new)), _on(self.device, free), self.lens, self.owned,
                      self.table, self.shared, self.free, self.used)
        p.check()
        self.lens, self.owned, self.shared, self.used = p.lens, p.owned, p.shared, p.free_used
        self._rows.update(zip(new, free))

    def compact(self) -> torch.Tensor:
        """Moves the held pages to the pool's front and returns their number
        (int32 [1] on the GPU): pages from there on are free."""
        self._between_steps()
        p = page_compact(self.k, self.v, self.owned, self.table, self.shared)
        self.table, self.shared, self.free, self.used = p.block_table, p.shared, p.free_pages, p.free_used
        return self.used

    def _planned(self, new: dict) -> PagePlan:
        counts, parents = [0] * self.max_requests, []
        tree = any(not isinstance(x, int) for x in new.values())
        for rid, x in new.items():
            counts[self._rows[rid]] = x if isinstance(x, int) else len(x)
        by_row = sorted(new, key=self._rows.get)
        if tree:
            for rid in by_row:
                x = new[rid]
                parents += list(range(-1, x - 1)) if isinstance(x, int) else [int(a) for a in x]
        most = max(counts)
        if tree and most > MAX_NODES:
            raise ValueError(f"{most} drafted tokens for a request (at most {MAX_NODES})")
        dev = self.device
        self._new, self._live, self._most, self._parents = counts, sum(x > 0 for x in counts), most, parents
        return page_plan(self.lens, _on(dev, counts), self.owned, self.table, self.free, self.used, self.page_size,
                         sum(counts), _on(dev, parents) if tree else None,
                         n_words=max(1, -(-most // 64)) if tree else 1)

    def begin(self, new: dict, check: bool = True, chunks: bool = False) -> PagePlan:
        """Plans a step.  new: request -> its number of new tokens (a chain),
        or the list of its drafted tokens' parents (-1: a child of the last
        committed token).  check: wait for the plan and raise OutOfPages if a
        request was refused; False leaves that to the caller (plan.status).
        chunks: chains may have more than 256 tokens (chunks of prompts); then no
        request of the step brings a tree."""
        if self._plan is not None:
            raise RuntimeError("a step has begun: commit it first")
        if chunks and any(not isinstance(x, int) for x in new.values()):
            raise ValueError("a step of chunks has no trees")
        if not chunks and any((x if isinstance(x, int) else len(x)) > MAX_NODES for x in new.values()):
            raise ValueError(f"at most {MAX_NODES} new tokens a request")
        if any(isinstance(x, int) and x < 0 for x in new.values()):
            raise ValueError("a negative number of new tokens")
        plan = self._planned(new)
        if check:
            plan.check()
        self._plan, self._checked = plan, check
        return plan

    def step(self, layer: int, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
             out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """One layer of the step: q [n_tokens, n_heads, d] (f32, or the cache's
        16-bit type; turned in place when rope=True), k_new, v_new
        [n_tokens, n_kv, d] of q's type.  Returns the attention output, in
        q's type."""
        if self._plan is None:
            raise RuntimeError("no step has begun")
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} out of range")
        p = self._plan
        paged_append(q, k_new, v_new, p.slots, p.positions if self.rope else None, self.k[layer], self.v[layer],
                     theta=self.theta, stream=stream)
        if self._most > MAX_NODES:
            return chunk_attention(q, self.k[layer], self.v[layer], self.table, p.kv_lens, p.node_start, scale=self.scale,
                                   out=out, stream=stream, n_live=self._live, max_new=self._most)
        return tree_attention(q, self.k[layer], self.v[layer], self.table, p.kv_lens, p.node_start, mask=p.mask,
                              scale=self.scale, out=out, stream=stream, n_live=self._live, max_new=self._most)

    def commit(self, paths: dict | None = None) -> None:
        """Ends the step.  paths: request -> the accepted nodes, in order
        (strictly increasing; [] for none of them); a request that is not named,
        or whose path is None, keeps all its new tokens (right for chains)."""
        if self._plan is None:
            raise RuntimeError("no step has begun")
        p, paths = self._plan, paths or {}
        want = {self._rows[r]: [int(a) for a in x] for r, x in paths.items() if x is not None}
        for row, x in want.items():
            if any(b <= a for a, b in zip([-1] + x, x)) or (x and x[-1] >= self._new[row]):
                raise ValueError(f"path {x} is not strictly increasing below {self._new[row]}")
        full = [want.get(r, list(range(t))) for r, t in enumerate(self._new)]
        wide = max(1, max(len(x) for x in full))
        dev = self.device
        path, count = _on(dev, [x + [0] * (wide - len(x)) for x in full]), _on(dev, [len(x) for x in full])
        self.lens = paged_commit(self.k, self.v, self.table, self.lens, p.kv_lens, p.node_start, path, count)
        self.owned, self.used = p.owned, p.free_used
        self._plan = None

    def verify(self, target: torch.Tensor, draft: torch.Tensor | None, tokens: torch.Tensor, u: torch.Tensor,
               u_next: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Ends a step of drafts with the paths that the target's probabilities
        keep (verify_drafts), without waiting for the GPU.  The first token of each
        request is its pending one, the others hang below it.  target, draft
        [n_tokens, vocab], tokens int32, u f32 [n_tokens]: by token row; u_next f32
        [max_requests]: by the requests' places.  Returns path, n_accept and the
        next tokens, by place (place(rid)); idle places, and requests that a plan
        begun without check refused, have n_accept 0 and next -1."""
        if self._plan is None:
            raise RuntimeError("no step has begun")
        p, most = self._plan, max(1, self._most)
        if most > MAX_NODES:
            raise ValueError(f"{most} tokens for a request (at most {MAX_NODES} can be verified)")
        parents = self._parents if p.mask is not None else [a - 1 for t in self._new for a in range(t)]
        path, count, token = verify_drafts(target, draft, tokens, _on(self.device, parents), p.node_start, u, u_next,
                                           max_path=most)
        if not self._checked:  # a refused request has token rows, but attention left them zero
            refused = p.status != 0
            path.masked_fill_(refused[:, None], -1)
            count.masked_fill_(refused, 0)
            token.masked_fill_(refused, -1)
        self.lens = paged_commit(self.k, self.v, self.table, self.lens, p.kv_lens, p.node_start, path, count)
        self.owned, self.used = p.owned, p.free_used
        self._plan = None
        return path, count, token

    def place(self, rid) -> int:
        """The request's row in the batch's tables."""
        return self._rows[rid]

    def cache(self, rid, layer: int):
        """(K, V) copies [length, n_kv, d] of a request's layer, in position
        order.  Waits for the GPU."""
        row, n = self._rows[rid], self.length(rid)
        pages = self.table[row, :-(-n // self.page_size)].long()
        return tuple(x[layer][pages].flatten(0, 1)[:n] for x in (self.k, self.v))
