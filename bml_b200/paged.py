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
  tree_attention  attention of the new tokens               (every layer)
  paged_commit    the accepted path moved to the front      (once a step)

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


class OutOfPages(RuntimeError):
    """A plan that refused a request (its status says why)."""


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
        "bml_paged_plan", "bml_paged_append", "bml_attn_tree_sized", "bml_paged_commit", "bml_attn_tree_workspace_size")))
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


class PagedBatcher:
    """DecodeBatcher over a paged cache, with drafts: requests join and leave
    between steps, a step brings each request any number of new tokens -- one
    to decode, a chain, or a tree of drafted tokens -- and commit() keeps the
    accepted ones.

    Per step: ``begin(new)`` plans it; for every layer ``step(layer, q, k, v)``
    stores the tokens and returns their attention; ``commit(paths)`` ends it.
    Token rows are the requests' tokens in the order of ``active``."""

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
        self._rows: dict = {}    # request -> its row of the tables
        self._plan = None        # of the step that has begun
        self._new = None         # new tokens of each row (host),
        self._live = self._most = 0  # how many rows have some, the most of one

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

    def remove(self, rid) -> None:
        """Drops a request and returns its pages.  Waits for the GPU."""
        if self._plan is not None:
            raise RuntimeError("a step has begun: commit it first")
        row = self._rows.pop(rid)
        n, used = int(self.owned[row]), int(self.used)
        self.free[used - n:used] = self._held(row, n)
        self.used = self.used - n
        self.owned[row] = 0
        self.lens[row] = 0

    def _held(self, row: int, n: int) -> torch.Tensor:
        """The row's pages moved to the end of the taken part of the free
        list: the list holds each page once, so those pages swap places with
        the ones that lie there."""
        pages = self.table[row, :n].clone()
        used = int(self.used)
        taken = self.free[:used]
        keep = taken[~torch.isin(taken, pages)]
        self.free[:used - n] = keep
        return pages

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
        self._new, self._live, self._most = counts, sum(x > 0 for x in counts), most
        return page_plan(self.lens, torch.tensor(counts, dtype=torch.int32, device=dev), self.owned, self.table,
                         self.free, self.used, self.page_size, sum(counts),
                         torch.tensor(parents, dtype=torch.int32, device=dev) if tree else None,
                         n_words=max(1, -(-most // 64)) if tree else 1)

    def begin(self, new: dict, check: bool = True) -> PagePlan:
        """Plans a step.  new: request -> its number of new tokens (a chain),
        or the list of its drafted tokens' parents (-1: a child of the last
        committed token).  check: wait for the plan and raise OutOfPages if a
        request was refused; False leaves that to the caller (plan.status)."""
        if self._plan is not None:
            raise RuntimeError("a step has begun: commit it first")
        if any((x if isinstance(x, int) else len(x)) > MAX_NODES for x in new.values()):
            raise ValueError(f"at most {MAX_NODES} new tokens a request")
        if any(isinstance(x, int) and x < 0 for x in new.values()):
            raise ValueError("a negative number of new tokens")
        plan = self._planned(new)
        if check:
            plan.check()
        self._plan = plan
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
        path = torch.tensor([x + [0] * (wide - len(x)) for x in full], dtype=torch.int32, device=dev)
        count = torch.tensor([len(x) for x in full], dtype=torch.int32, device=dev)
        self.lens = paged_commit(self.k, self.v, self.table, self.lens, p.kv_lens, p.node_start, path, count)
        self.owned, self.used = p.owned, p.free_used
        self._plan = None

    def cache(self, rid, layer: int):
        """(K, V) copies [length, n_kv, d] of a request's layer, in position
        order.  Waits for the GPU."""
        row, n = self._rows[rid], self.length(rid)
        pages = self.table[row, :-(-n // self.page_size)].long()
        return tuple(x[layer][pages].flatten(0, 1)[:n] for x in (self.k, self.v))
