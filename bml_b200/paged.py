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
from dataclasses import dataclass

import torch

from . import _lib as L
from .attention import _need, _ptr, _stream, dtype_code
from .batching import MAX_PENDING_REQUESTS, AtCapacity

MAX_NODES = 256  # drafted tokens of one request in tree_attention
PLAN_NO_PAGES, PLAN_BAD, PLAN_NO_ROOM = 1, 2, 4  # status values of a plan


class OutOfPages(RuntimeError):
    """A plan that refused a request (its status says why)."""


def _arg(t, name: str, dtype, shape=None, device=None) -> None:
    _need(t, name, dtype)
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


class _On:
    """Makes a call's device current, and its stream where one is given, so
    that the buffers it allocates belong to the stream that uses them."""

    def __init__(self, device: torch.device, stream=None):
        if stream is not None and stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
        self._ctx = torch.cuda.stream(stream) if stream is not None else torch.cuda.device(device)

    def __enter__(self):
        self._ctx.__enter__()
        return _stream()

    def __exit__(self, *exc):
        return self._ctx.__exit__(*exc)


@dataclass
class PagePlan:
    """One step's plan; all tensors on the device (see bml_paged_plan)."""
    node_start: torch.Tensor  # int32 [n + 1]
    kv_lens: torch.Tensor     # int32 [n]
    owned: torch.Tensor       # int32 [n]
    free_used: torch.Tensor   # int32 [1]
    slots: torch.Tensor       # int64 [n_tokens]
    positions: torch.Tensor   # int32 [n_tokens]
    status: torch.Tensor      # int32 [n]
    mask: torch.Tensor | None  # int64 [n_tokens, n_words], with parents

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
    _arg(lens, "lens", torch.int32)
    if lens.dim() != 1:
        raise ValueError("lens must have 1 dim")
    n, dev = lens.shape[0], lens.device
    _arg(n_new, "n_new", torch.int32, (n,), dev)
    _arg(owned, "owned", torch.int32, (n,), dev)
    _arg(block_table, "block_table", torch.int32, None, dev)
    if block_table.dim() != 2 or block_table.shape[0] != n:
        raise ValueError(f"block_table must be [{n}, max_pages], got {tuple(block_table.shape)}")
    _arg(free_pages, "free_pages", torch.int32, None, dev)
    if free_pages.dim() != 1:
        raise ValueError("free_pages must have 1 dim")
    _arg(free_used, "free_used", torch.int32, (1,), dev)
    if n_tokens < 0:
        raise ValueError("n_tokens must not be negative")
    if parents is not None:
        _arg(parents, "parents", torch.int32, (n_tokens,), dev)
        if not 1 <= n_words <= MAX_NODES // 64:
            raise ValueError(f"n_words must be 1 to {MAX_NODES // 64}, got {n_words}")
    with _On(dev, stream) as st:
        i32 = dict(dtype=torch.int32, device=dev)
        p = PagePlan(torch.empty(n + 1, **i32), torch.empty(n, **i32), torch.empty(n, **i32), torch.empty(1, **i32),
                     torch.empty(n_tokens, dtype=torch.int64, device=dev), torch.empty(n_tokens, **i32),
                     torch.empty(n, **i32),
                     None if parents is None else torch.empty(n_tokens, n_words, dtype=torch.int64, device=dev))
        L.call("bml_paged_plan", _ptr(lens), _ptr(n_new), _ptr(owned), n, _ptr(free_pages), free_pages.numel(),
               _ptr(free_used), page_size, block_table.shape[1], _ptr(block_table),
               None if parents is None else _ptr(parents), n_tokens, n_words, _ptr(p.node_start), _ptr(p.kv_lens),
               _ptr(p.owned), _ptr(p.free_used), _ptr(p.slots), _ptr(p.positions),
               None if p.mask is None else _ptr(p.mask), _ptr(p.status), st)
    return p


def _pools(k_pool, v_pool, ndim: int, device=None):
    _need(k_pool, "k_pool", None, ndim)
    _need(v_pool, "v_pool", k_pool.dtype, ndim)
    if k_pool.shape != v_pool.shape or k_pool.device != v_pool.device:
        raise ValueError(f"k_pool {tuple(k_pool.shape)} and v_pool {tuple(v_pool.shape)} do not match")
    if device is not None and k_pool.device != device:
        raise ValueError(f"the pools are on {k_pool.device}, expected {device}")


def paged_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
                 positions: torch.Tensor | None, k_pool: torch.Tensor, v_pool: torch.Tensor,
                 q_out: torch.Tensor | None = None, theta: float = 10000.0, stream=None) -> torch.Tensor | None:
    """RoPE and store of one layer's new tokens: q [n, n_heads, d] turned by
    positions [n] int32 (in place, or into q_out), k turned and v as is
    ([n, n_kv, d]) into row slots[t] (int64) of the pools
    [n_pages, page_size, n_kv, d].  q, k, v in one type (f32, f16, bf16), the
    pools in any.  positions None: no rotation; q None: no queries.  A token
    whose slot is -1 (or outside the pool) is skipped.  Returns the turned q."""
    _need(k, "k", None, 3)
    _need(v, "v", k.dtype, 3)
    n, n_kv, d = k.shape
    dev = k.device
    if k.shape != v.shape or v.device != dev:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    _pools(k_pool, v_pool, 4, dev)
    if tuple(k_pool.shape[2:]) != (n_kv, d):
        raise ValueError(f"pool rows {tuple(k_pool.shape[2:])} do not match k {tuple(k.shape)}")
    _arg(slots, "slots", torch.int64, (n,), dev)
    if positions is not None:
        _arg(positions, "positions", torch.int32, (n,), dev)
    n_heads = 0
    if q is not None:
        _arg(q, "q", k.dtype, None, dev)
        if q.dim() != 3 or q.shape[0] != n or q.shape[2] != d:
            raise ValueError(f"q {tuple(q.shape)} does not match k {tuple(k.shape)}")
        n_heads = q.shape[1]
        if q_out is None:
            q_out = q
        else:
            _arg(q_out, "q_out", q.dtype, q.shape, dev)
    elif q_out is not None:
        raise ValueError("q_out without q")
    with _On(dev, stream) as st:
        L.call("bml_paged_append", None if q is None else _ptr(q), _ptr(k), _ptr(v), dtype_code(k.dtype), _ptr(slots),
               None if positions is None else _ptr(positions), n, n_heads, n_kv, d, float(theta),
               None if q is None else _ptr(q_out), _ptr(k_pool), _ptr(v_pool), dtype_code(k_pool.dtype),
               k_pool.shape[0] * k_pool.shape[1], st)
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
                   stream=None) -> torch.Tensor:
    """Attention of every request's new tokens over its pages.  q
    [n_tokens, n_heads, d] holds request i's T tokens in rows
    node_start[i]..node_start[i+1]; a token attends over the request's first
    kv_lens[i] - T positions and over the new tokens that its mask row
    (int64 [n_tokens, 1 to 4], bit j: the request's j-th new token) names;
    without a mask, over itself and those before it (T = 1: plain decode).
    q is f32, or of the pools' 16-bit type; the result has q's type.  At most
    256 new tokens a request (64 a mask word).  Rows that see nothing, and
    those of requests that page_plan refused, are zero.  scale < 0 selects
    1/sqrt(d).

    workspace: an uint8 tensor of tree_workspace_size bytes for calls that
    must not allocate; calls that share one must not overlap.  By default
    scratch comes from torch's allocator, on the call's stream."""
    _need(q, "q", None, 3)
    n_tokens, n_heads, d = q.shape
    dev = q.device
    _pools(k_pool, v_pool, 4, dev)
    if k_pool.shape[3] != d:
        raise ValueError(f"q {tuple(q.shape)} does not match the pools {tuple(k_pool.shape)}")
    n = kv_lens.shape[0] if isinstance(kv_lens, torch.Tensor) and kv_lens.dim() == 1 else -1
    _arg(kv_lens, "kv_lens", torch.int32, (n,), dev)
    _arg(node_start, "node_start", torch.int32, (n + 1,), dev)
    _arg(block_table, "block_table", torch.int32, None, dev)
    if block_table.dim() != 2 or block_table.shape[0] != n:
        raise ValueError(f"block_table must be [{n}, max_pages], got {tuple(block_table.shape)}")
    n_words = 0
    if mask is not None:
        _arg(mask, "mask", torch.int64, None, dev)
        if mask.dim() != 2 or mask.shape[0] != n_tokens or not 1 <= mask.shape[1] <= MAX_NODES // 64:
            raise ValueError(f"mask must be [{n_tokens}, 1 to {MAX_NODES // 64}], got {tuple(mask.shape)}")
        n_words = mask.shape[1]
    with _On(dev, stream) as st:
        if out is None:
            out = torch.empty_like(q)
        else:
            _arg(out, "out", q.dtype, q.shape, dev)
        if workspace is None:
            workspace = torch.empty(tree_workspace_size(d, dev), dtype=torch.uint8, device=dev)
        else:
            _arg(workspace, "workspace", torch.uint8, None, dev)
        L.call("bml_attn_tree", _ptr(q), dtype_code(q.dtype), n_tokens, n_heads, k_pool.shape[2], d, _ptr(k_pool),
               _ptr(v_pool), dtype_code(k_pool.dtype), k_pool.shape[0], k_pool.shape[1], _ptr(block_table),
               block_table.shape[1], _ptr(kv_lens), _ptr(node_start), n, None if mask is None else _ptr(mask), n_words,
               float(scale), _ptr(out), _ptr(workspace), workspace.numel(), st)
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
    _pools(k_pools, v_pools, 5)
    dev = k_pools.device
    n = lens.shape[0] if isinstance(lens, torch.Tensor) and lens.dim() == 1 else -1
    _arg(lens, "lens", torch.int32, (n,), dev)
    _arg(kv_lens, "kv_lens", torch.int32, (n,), dev)
    _arg(node_start, "node_start", torch.int32, (n + 1,), dev)
    _arg(n_accept, "n_accept", torch.int32, (n,), dev)
    _arg(block_table, "block_table", torch.int32, None, dev)
    _arg(path, "path", torch.int32, None, dev)
    if block_table.dim() != 2 or block_table.shape[0] != n:
        raise ValueError(f"block_table must be [{n}, max_pages], got {tuple(block_table.shape)}")
    if path.dim() != 2 or path.shape[0] != n:
        raise ValueError(f"path must be [{n}, max_path], got {tuple(path.shape)}")
    layers, n_pages, page_size, n_kv, d = k_pools.shape
    with _On(dev, stream) as st:
        new = torch.empty_like(lens)
        L.call("bml_paged_commit", _ptr(k_pools), _ptr(v_pools), layers, n_pages, page_size, n_kv, d,
               dtype_code(k_pools.dtype), _ptr(block_table), block_table.shape[1], _ptr(lens), _ptr(kv_lens),
               _ptr(node_start), n, _ptr(path), path.shape[1], _ptr(n_accept), _ptr(new), st)
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
        self._new = None         # new tokens of each row (host)

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
        except OutOfPages:
            del self._rows[rid]
            raise
        for layer in range(self.n_layers):
            paged_append(None, k_prompt[layer].contiguous(), v_prompt[layer].contiguous(), plan.slots, None,
                         self.k[layer], self.v[layer])
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
        self._new = counts
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
                              scale=self.scale, out=out, stream=stream)

    def commit(self, paths: dict | None = None) -> None:
        """Ends the step.  paths: request -> the accepted nodes, in order
        (strictly increasing); a request that is not named, or None, keeps
        all its new tokens (right for chains)."""
        if self._plan is None:
            raise RuntimeError("no step has begun")
        p, paths = self._plan, paths or {}
        want = {self._rows[r]: [int(a) for a in x] for r, x in paths.items()}
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
