"""Cases of the paged-cache operators: page planning, RoPE append into pages,
attention of drafted-token trees over pages, and the commit of an accepted
path.

`run` computes an operator in its plain form (elementary torch operations in
32 bits) where `own` is false, and calls the package's entry points where it
is true.  `exact` is the definition in 64 bits, one request at a time."""
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One request in the middle of a chat on the TinyLlama shape, a draft of
        # eight tokens: the smallest call, where latency counts.
        dict(name="tree-chat", op="attention", n=1, len_lo=700, len_hi=700, node_lo=8, node_hi=8, heads=32, kv=4,
             dim=64, q="f16", cache="f16", page=16, tree=True, shape=1),
        # A server's batch on the Llama-3 shape, drafts of 16 to 64 tokens.
        dict(name="tree-batch", op="attention", n=32, len_lo=1024, len_hi=8192, node_lo=16, node_hi=64, heads=32, kv=8,
             dim=128, q="bf16", cache="bf16", page=64, tree=True, shape=2),
        # One long document with a wide draft.
        dict(name="tree-long", op="attention", n=1, len_lo=131008, len_hi=131008, node_lo=64, node_hi=64, heads=32,
             kv=8, dim=128, q="bf16", cache="bf16", page=128, tree=True, shape=3),
        # The single-token form: a ragged batch that decodes without a draft.
        dict(name="decode-ragged", op="attention", n=64, len_lo=128, len_hi=4096, node_lo=1, node_hi=1, heads=32, kv=4,
             dim=64, q="f16", cache="f16", page=16, tree=False, shape=4),
        # The reference's own precision: 32-bit queries over a 32-bit cache.
        dict(name="tree-f32", op="attention", n=4, len_lo=500, len_hi=3001, node_lo=7, node_hi=25, heads=32, kv=8,
             dim=128, q="f32", cache="f32", page=32, tree=True, shape=5),
        # The batcher's form: 32-bit queries, 16-bit pages, one token a request.
        dict(name="decode-f32-queries", op="attention", n=32, len_lo=1000, len_hi=4096, node_lo=1, node_hi=1, heads=32,
             kv=8, dim=128, q="f32", cache="bf16", page=64, tree=False, shape=6),
        # One decode step's plan of a few requests with drafts.
        dict(name="plan-drafts", op="plan", n=16, len_lo=100, len_hi=4000, new_lo=1, new_hi=63, page=16, tree=True,
             words=1, shape=7),
        # Admission of many prompts at once.
        dict(name="plan-prompts", op="plan", n=512, len_lo=0, len_hi=64, new_lo=17, new_hi=4096, page=64, tree=False,
             words=0, shape=8),
        # One layer's append of a small batch's drafted tokens, from 32-bit projections.
        dict(name="append-drafts", op="append", tokens=37, heads=32, kv=4, dim=64, src="f32", cache="f16", page=16,
             far=2048, shape=9),
        # One layer's append of prompts, far into a long context.
        dict(name="append-prompts", op="append", tokens=16001, heads=32, kv=8, dim=128, src="bf16", cache="bf16",
             page=64, far=131072, shape=10),
        # One request's accepted path over every layer of the TinyLlama shape.
        dict(name="commit-chat", op="commit", n=1, len_lo=700, len_hi=700, node_lo=8, node_hi=8, layers=22, kv=4,
             dim=64, cache="f16", page=16, shape=11),
        # A batch's accepted paths over every layer of the Llama-3 shape.
        dict(name="commit-batch", op="commit", n=64, len_lo=100, len_hi=900, node_lo=16, node_hi=64, layers=32, kv=8,
             dim=128, cache="bf16", page=64, shape=12),
    ]


HEADS = [(8, 2, 64), (12, 4, 64), (32, 4, 64), (20, 4, 128), (16, 16, 128), (32, 8, 128), (64, 8, 128)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "plan", "append", "commit"])
    shape, page = rng.randrange(1, 1 << 30), rng.choice([16, 32, 64, 128])
    if op == "attention":
        heads, kv, dim = rng.choice(HEADS)
        q, cache = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f16"), ("f32", "f32"),
                               ("f32", "bf16"), ("f32", "f16")])
        n = _log(rng, 1, 64)
        tree = rng.random() < 0.7
        # positions x nodes x heads x dim stay well below the largest listed case's
        node_hi = _log(rng, 1, 160) if tree else 1
        room = 110000 if q != "f32" else 30000
        hi = max(1, min(room, 131008 * 40 // node_hi * 32 // heads) // n)
        hi = _log(rng, min(hi, 24), hi)
        return dict(op=op, n=n, len_lo=rng.choice([0, 1, hi // 3, hi]), len_hi=hi, node_lo=rng.choice([1, node_hi]),
                    node_hi=node_hi, heads=heads, kv=kv, dim=dim, q=q, cache=cache, page=page, tree=tree, shape=shape)
    if op == "plan":
        tree = rng.random() < 0.5
        n = _log(rng, 1, 512)
        words = rng.choice([1, 1, 2, 4]) if tree else 0
        return dict(op=op, n=n, len_lo=0, len_hi=_log(rng, 16, 8000), new_lo=rng.choice([0, 1]),
                    new_hi=_log(rng, 1, 64 * words if tree else 4000), page=page, tree=tree, words=words, shape=shape)
    if op == "append":
        heads, kv, dim = rng.choice(HEADS)
        src, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16"),
                                 ("bf16", "f32")])
        return dict(op=op, tokens=_log(rng, 1, 4000), heads=heads, kv=kv, dim=dim, src=src, cache=cache, page=page,
                    far=_log(rng, 64, 131072), shape=shape)
    heads, kv, dim = rng.choice(HEADS)
    return dict(op=op, n=_log(rng, 1, 48), len_lo=0, len_hi=_log(rng, 16, 800), node_lo=2, node_hi=_log(rng, 2, 64),
                layers=_log(rng, 1, 32), kv=min(kv, 8), dim=dim, cache=rng.choice(["f32", "bf16", "f16"]), page=page,
                shape=shape)


def _sizes(case):
    """The ragged sizes of a case, the same for every seed."""
    r = random.Random(case["shape"])
    if case["op"] == "append":
        return None
    lens = [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["n"])]
    lo, hi = (case["new_lo"], case["new_hi"]) if case["op"] == "plan" else (case["node_lo"], case["node_hi"])
    new = [r.randint(lo, hi) for _ in range(case["n"])]
    accept = [r.randint(1, max(1, min(8, t - 1))) if t > 1 else 0 for t in new]
    return lens, new, accept


def work(case):
    if case["op"] == "append":
        n, row = case["tokens"], case["kv"] * case["dim"]
        q = case["heads"] * case["dim"]
        s, c = SIZE[case["src"]], SIZE[case["cache"]]
        return {"bytes": n * (2 * q * s + 2 * row * s + 2 * row * c + 12), "flops": n * 3 * (q + row)}
    lens, new, accept = _sizes(case)
    ps = case["page"]
    if case["op"] == "attention":
        row, h = case["kv"] * case["dim"], case["heads"] * case["dim"]
        c, s = SIZE[case["cache"]], SIZE[case["q"]]
        pages = sum(-(-(a + b) // ps) for a, b in zip(lens, new))
        words = _words(new) if case["tree"] else 0
        return {"bytes": sum(2 * row * c * (a + b) for a, b in zip(lens, new)) + sum(new) * (2 * h * s + 8 * words)
                + 4 * pages + 8 * len(lens),
                "flops": sum(4 * h * b * (a + b) for a, b in zip(lens, new))}
    if case["op"] == "plan":
        held = sum(-(-a // ps) for a in lens)
        pages = sum(-(-(a + b) // ps) for a, b in zip(lens, new)) - held
        touched = sum(-(-(a + b) // ps) - a // ps for a, b in zip(lens, new) if b)
        return {"bytes": sum(new) * (12 + ((4 + 8 * case["words"]) if case["tree"] else 0)) + 8 * pages + 4 * touched
                + 28 * len(lens), "flops": 0}
    return {"bytes": sum(accept) * case["layers"] * case["kv"] * case["dim"] * SIZE[case["cache"]] * 4
            + 16 * len(lens) + 4 * sum(accept), "flops": 0}


def _words(new):
    return max(1, -(-max(new) // 64))


# ---------------------------------------------------------------------------
# What a user's program holds
# ---------------------------------------------------------------------------
def _ints(v, dev="cuda", dt=torch.int32):
    return torch.tensor(v, dtype=dt, device=dev)


def _starts(new):
    out = [0]
    for b in new:
        out.append(out[-1] + b)
    return out


def _parents(new, g):
    """Random drafts: node j hangs below one of the nodes before it, or below
    the last committed token (-1); most below a recent one."""
    total = sum(new)
    j = torch.cat([torch.arange(b) for b in new]) if total else torch.zeros(0, dtype=torch.long)
    back = 1 + (torch.rand(total, generator=g) ** 2 * 6).long()
    return (j - back).clamp_(min=-1).to(torch.int32)


def _table(lens, new, page, g, spare=3):
    """Block tables over a shuffled pool: pages for every position."""
    need = [-(-(a + b) // page) for a, b in zip(lens, new)]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    return table.cuda(), n_pages


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gc = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dt):
        return torch.randn(shape, generator=gc, device="cuda", dtype=torch.float32).to(DT[dt])

    s = {"case": case}
    if case["op"] == "append":
        n, kv, d = case["tokens"], case["kv"], case["dim"]
        n_pages = -(-n // case["page"]) + 4
        s["q"] = normal((n, case["heads"], d), case["src"])
        s["k"], s["v"] = normal((n, kv, d), case["src"]), normal((n, kv, d), case["src"])
        s["k_pool"] = normal((n_pages, case["page"], kv, d), case["cache"])
        s["v_pool"] = normal((n_pages, case["page"], kv, d), case["cache"])
        s["q_out"] = torch.empty_like(s["q"])
        # a run of consecutive positions on shuffled pages, as a prompt has
        pages = torch.randperm(n_pages, generator=g)
        t = torch.arange(n) + 3
        s["slots"] = (pages[t // case["page"]] * case["page"] + t % case["page"]).cuda()
        s["positions"] = ((t + int(torch.randint(0, case["far"], (1,), generator=g))) % case["far"]).to(
            torch.int32).cuda()
        return s
    lens, new, accept = _sizes(case)
    s["node_start"] = _ints(_starts(new))
    if case["op"] == "attention":
        kv, d = case["kv"], case["dim"]
        s["table"], n_pages = _table(lens, new, case["page"], g)
        s["k_pool"] = normal((n_pages, case["page"], kv, d), case["cache"])
        s["v_pool"] = normal((n_pages, case["page"], kv, d), case["cache"])
        s["q"] = normal((sum(new), case["heads"], d), case["q"])
        s["kv_lens"] = _ints([a + b for a, b in zip(lens, new)])
        s["mask"] = None
        if case["tree"]:
            s["mask"] = _masks(_parents(new, g).cuda(), s["node_start"], max(new), _words(new))[0]
        return s
    if case["op"] == "plan":
        held = [-(-a // case["page"]) for a in lens]
        need = [-(-(a + b) // case["page"]) for a, b in zip(lens, new)]
        n_pages = sum(need) + 5
        order = torch.randperm(n_pages, generator=g).to(torch.int32)
        table = torch.full((case["n"], max(need) + 1), -1, dtype=torch.int32)
        at = 0
        for i, k in enumerate(held):
            table[i, :k] = order[at:at + k]
            at += k
        s["table"], s["free"], s["used"] = table.cuda(), order.cuda(), _ints([at])
        s["lens"], s["new"], s["owned"] = _ints(lens), _ints(new), _ints(held)
        s["parents"] = _parents(new, g).cuda() if case["tree"] else None
        s["tokens"] = sum(new)
        return s
    kv, d, layers = case["kv"], case["dim"], case["layers"]
    s["table"], n_pages = _table(lens, new, case["page"], g)
    s["k_pool"] = normal((layers, n_pages, case["page"], kv, d), case["cache"])
    s["v_pool"] = normal((layers, n_pages, case["page"], kv, d), case["cache"])
    s["lens"], s["kv_lens"] = _ints(lens), _ints([a + b for a, b in zip(lens, new)])
    path = torch.zeros(len(lens), 8, dtype=torch.int32)
    for i, (t, a) in enumerate(zip(new, accept)):
        if a:
            path[i, :a] = (1 + torch.randperm(t - 1, generator=g)[:a]).sort().values.to(torch.int32)
    s["path"], s["accept"] = path.cuda(), _ints(accept)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        import bml_b200
        if case["op"] == "attention":
            return bml_b200.tree_attention(s["q"], s["k_pool"], s["v_pool"], s["table"], s["kv_lens"], s["node_start"],
                                           mask=s["mask"])
        if case["op"] == "append":
            q = bml_b200.paged_append(s["q"], s["k"], s["v"], s["slots"], s["positions"], s["k_pool"], s["v_pool"],
                                      q_out=s["q_out"])
            return q, s["k_pool"], s["v_pool"]
        if case["op"] == "plan":
            p = bml_b200.page_plan(s["lens"], s["new"], s["owned"], s["table"], s["free"], s["used"], case["page"],
                                   s["tokens"], parents=s["parents"], n_words=case["words"])
            return _plan_outputs(s, p.node_start, p.kv_lens, p.owned, p.free_used, p.slots, p.positions, p.mask,
                                 p.status)
        new_lens = bml_b200.paged_commit(s["k_pool"], s["v_pool"], s["table"], s["lens"], s["kv_lens"],
                                         s["node_start"], s["path"], s["accept"])
        return new_lens, s["k_pool"], s["v_pool"]
    return {"attention": _attention, "append": _append, "plan": _plan, "commit": _commit}[case["op"]](s)


def _plan_outputs(s, starts, kv_lens, owned, used, slots, positions, mask, status):
    out = [s["table"], starts, kv_lens, owned, used, slots, positions, status]
    return out + [mask] if mask is not None else out


def _attention(s):
    q, mask, start = s["q"], s["mask"], s["node_start"].long()
    kv, d = s["k_pool"].shape[2:]
    ps = s["k_pool"].shape[1]
    case = s["case"]
    t_max = case["node_hi"]
    heads, group = q.shape[1], q.shape[1] // kv
    total = s["kv_lens"].long()
    nodes = start[1:] - start[:-1]
    pos = torch.arange(s["table"].shape[1] * ps, device=q.device)
    rows = (s["table"].long()[:, pos // ps] * ps + pos % ps).clamp(min=0)
    k = s["k_pool"].reshape(-1, kv, d)[rows].float()              # [n, L, kv, d]
    v = s["v_pool"].reshape(-1, kv, d)[rows].float()
    t = torch.arange(t_max, device=q.device)
    tok = (start[:-1, None] + t).clamp(max=max(0, q.shape[0] - 1))   # [n, T]
    here = t < nodes[:, None]
    qs = q.float()[tok].reshape(len(total), t_max, kv, group, d)
    node = pos - (total - nodes)[:, None]                         # [n, L]: which drafted node a position is
    if mask is None:
        seen = node[:, None, :] <= t[:, None]
    else:
        word = mask[tok]                                          # [n, T, W]
        at = node.clamp(min=0)[:, None, :].expand(-1, t_max, -1)
        bits = torch.gather(word, 2, (at // 64).clamp(max=word.shape[2] - 1))
        seen = (node[:, None, :] < 0) | (((bits >> (at % 64)) & 1) == 1)
    seen = seen & (pos < total[:, None])[:, None, :] & here[:, :, None]
    sc = torch.einsum("ntkgd,nlkd->nkgtl", qs, k) * (1.0 / d ** 0.5)
    see = seen[:, None, None]
    sc = torch.where(see, sc, torch.full_like(sc, float("-inf")))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top.isinf(), torch.zeros_like(top), top))
    l = p.sum(-1, keepdim=True)
    v = torch.where((pos < total[:, None])[:, :, None, None], v, torch.zeros_like(v))
    o = torch.einsum("nkgtl,nlkd->ntkgd", p / torch.where(l > 0, l, torch.ones_like(l)), v)
    out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    out[tok[here]] = o.reshape(len(total), t_max, heads, d)[here]
    return out.to(q.dtype)


def _turn(x, cos, sin):
    """Interleaved pairs of the last dimension turned by their angles."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _angles(positions, d):
    i = torch.arange(0, d, 2, device=positions.device, dtype=torch.float64)
    return positions.double()[:, None] * 10000.0 ** (-i / d)


def _append(s):
    kv, d = s["k_pool"].shape[2:]
    a = _angles(s["positions"], d)
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    q = _turn(s["q"].float(), cos, sin).to(s["q"].dtype)
    kt = _turn(s["k"].float(), cos, sin)
    s["k_pool"].view(-1, kv, d)[s["slots"]] = kt.to(s["k_pool"].dtype)
    s["v_pool"].view(-1, kv, d)[s["slots"]] = s["v"].float().to(s["v_pool"].dtype)
    return q, s["k_pool"], s["v_pool"]


def _masks(parents, starts, t_max, words):
    """Ancestor bits [N, words] and depths [N] of drafts: a tree's closure is
    a power of its parent matrix (plus the identity)."""
    starts = starts.long()
    nodes = starts[1:] - starts[:-1]
    t_max = max(1, t_max)
    t = torch.arange(t_max, device=parents.device)
    here = t < nodes[:, None]
    if parents.numel() == 0:
        return (torch.zeros(0, words, dtype=torch.int64, device=parents.device),
                torch.zeros(0, dtype=torch.int32, device=parents.device))
    tok = (starts[:-1, None] + t).clamp(max=parents.shape[0] - 1)
    par = torch.where(here, parents.long()[tok], torch.full_like(tok, -1))
    up = (par[:, :, None] == t).double() + torch.eye(t_max, dtype=torch.float64, device=parents.device)
    seen = torch.linalg.matrix_power(up, t_max) > 0               # [n, T, T]
    seen = torch.cat((seen, seen.new_zeros(len(nodes), t_max, words * 64 - t_max)), 2) if words * 64 > t_max else seen
    bits = seen.view(len(nodes), t_max, words, 64).long() << torch.arange(64, device=parents.device)
    mask = torch.zeros(parents.shape[0], words, dtype=torch.int64, device=parents.device)
    depth = torch.zeros(parents.shape[0], dtype=torch.int32, device=parents.device)
    mask[tok[here]] = bits.sum(-1)[here]
    depth[tok[here]] = (seen.sum(-1) - 1).int()[here]
    return mask, depth


def _plan(s):
    ps, n_tok = s["case"]["page"], s["tokens"]
    lens, new, owned = s["lens"].long(), s["new"].long(), s["owned"].long()
    table, free = s["table"], s["free"]
    dev = lens.device
    need = (lens + new + ps - 1) // ps
    add = (need - owned).clamp(min=0)
    cum = add.cumsum(0)
    short = (add > 0) & (cum > free.numel() - s["used"])
    ends = new.cumsum(0)
    starts = torch.cat((ends.new_zeros(1), ends))
    first = s["used"] + cum - add
    p = torch.arange(table.shape[1], device=dev)
    fresh = (p >= owned[:, None]) & (p < need[:, None]) & ~short[:, None]
    got = free[(first[:, None] + p - owned[:, None]).clamp(0, free.numel() - 1)]
    table.copy_(torch.where(fresh, got, table))
    tok = torch.arange(n_tok, device=dev)
    req = torch.searchsorted(ends, tok, right=True).clamp(max=len(lens) - 1)
    pos = lens[req] + tok - starts[req]
    slots = table[req, pos // ps].long() * ps + pos % ps
    slots = torch.where(short[req], torch.full_like(slots, -1), slots)
    mask = None
    if s["parents"] is not None:
        mask, depth = _masks(s["parents"], starts, s["case"]["new_hi"], s["case"]["words"])
        pos = lens[req] + depth
    kv = torch.where(short, torch.zeros_like(lens), lens + new).int()
    held = torch.where(short, owned, torch.maximum(owned, need)).int()
    used = s["used"] + torch.where(short, torch.zeros_like(cum), cum).amax().int()
    return _plan_outputs(s, starts.int(), kv, held, used, slots, pos.int(), mask, short.int())


def _commit(s):
    ps = s["k_pool"].shape[2]
    lens, path, accept = s["lens"].long(), s["path"].long(), s["accept"].long()
    k = torch.arange(path.shape[1], device=lens.device)
    take = k < accept[:, None]
    req = torch.arange(len(lens), device=lens.device)[:, None].expand_as(path)[take]
    src, dst = (lens[:, None] + path)[take], (lens[:, None] + k)[take]
    table = s["table"].long()
    rows = [table[req, p // ps] * ps + p % ps for p in (src, dst)]
    kp, vp = (p.view(p.shape[0], -1, *p.shape[3:]) for p in (s["k_pool"], s["v_pool"]))
    kp[:, rows[1]] = kp[:, rows[0]]
    vp[:, rows[1]] = vp[:, rows[0]]
    return (lens + accept).int(), s["k_pool"], s["v_pool"]


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("plan", "commit"):  # whole numbers, and rows that only move
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        d = case["dim"]
        pos = s["positions"].to(torch.float64)
        freq = torch.exp(torch.arange(d // 2, dtype=torch.float64, device="cuda") * (-2.0 / d)
                         * torch.log(torch.tensor(10000.0, dtype=torch.float64)).item())
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda").expand(len(pos), d // 2).contiguous(),
                           pos[:, None] * freq)[:, None]

        def turned(x):
            z = torch.view_as_complex(x.double().reshape(*x.shape[:2], d // 2, 2).contiguous())
            return torch.view_as_real(z * turn).reshape(x.shape)

        kp, vp = s["k_pool"].double(), s["v_pool"].double()
        page, off = s["slots"] // case["page"], s["slots"] % case["page"]
        kp[page, off] = turned(s["k"])
        vp[page, off] = s["v"].double()
        return turned(s["q"]), kp, vp
    lens, new, _ = _sizes(case)
    group = case["heads"] // case["kv"]
    out, at = [], 0
    for i, (a, b) in enumerate(zip(lens, new)):
        pages = s["table"][i, :-(-(a + b) // case["page"])].long()
        k = s["k_pool"][pages].flatten(0, 1)[:a + b].double()
        v = s["v_pool"][pages].flatten(0, 1)[:a + b].double()
        q = s["q"][at:at + b].double()
        see = torch.ones(b, a + b, dtype=torch.bool, device="cuda")
        for t in range(b):
            for j in range(b):
                if s["mask"] is None:
                    if j > t:
                        see[t, a + j] = False
        if s["mask"] is not None:
            w = s["mask"][at:at + b]
            j = torch.arange(b, device="cuda")
            see[:, a:] = ((w[:, j // 64] >> (j % 64)) & 1).bool()
        for h in range(case["kv"]):
            x = torch.matmul(q[:, h * group:(h + 1) * group].transpose(0, 1), k[:, h].T) / case["dim"] ** 0.5
            x = torch.softmax(x.masked_fill(~see, float("-inf")), -1)
            out.append(torch.matmul(x, v[:, h]).transpose(0, 1))
        at += b
        heads = torch.cat(out[-case["kv"]:], 1)
        out[-case["kv"]:] = [heads]
    return torch.cat(out, 0)
