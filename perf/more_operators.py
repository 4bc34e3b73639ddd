"""Cases of the paged cache's serving operators: attention of prompt chunks of
any length over pages, verification of drafted tokens against the target's
probabilities, and forking, freeing and compacting pages.

`run` computes an operator in its plain form (elementary torch operations in
32 bits; sums over a vocabulary, which decide about whole numbers, in 64)
where `own` is false, and calls the package's entry points where it is true.
`exact` is the attention's definition in 64 bits, one request and head at a
time."""
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
        # One turn of a chat on the TinyLlama shape: the user's message joins the
        # cache in one chunk.  The smallest call, where latency counts.
        dict(name="chunk-chat", op="chunk", n=1, len_lo=700, len_hi=700, new_lo=300, new_hi=300, heads=32, kv=4, dim=64,
             q="f16", cache="f16", page=16, shape=1),
        # A server's mixed batch on the Llama-3 shape: requests that decode one
        # token beside others whose prompts come in chunks of up to 1000 tokens.
        dict(name="chunk-mixed", op="chunk", n=16, len_lo=100, len_hi=4096, new_lo=-1000, new_hi=1000, heads=32, kv=8,
             dim=128, q="bf16", cache="bf16", page=64, shape=2),
        # A chunk far into a long document.
        dict(name="chunk-long", op="chunk", n=1, len_lo=30720, len_hi=30720, new_lo=2048, new_hi=2048, heads=32, kv=8,
             dim=128, q="bf16", cache="bf16", page=128, shape=3),
        # The reference's own precision: fresh prompts in 32 bits.
        dict(name="chunk-f32", op="chunk", n=3, len_lo=0, len_hi=900, new_lo=257, new_hi=701, heads=32, kv=8, dim=128,
             q="f32", cache="f32", page=32, shape=4),
        # One request's draft of picked (not drawn) tokens over an odd vocabulary.
        dict(name="verify-chat", op="verify", n=1, new_lo=8, new_hi=8, vocab=32001, probs="f16", draft=False, shape=5),
        # A batch's drawn drafts over a large vocabulary.
        dict(name="verify-batch", op="verify", n=48, new_lo=2, new_hi=32, vocab=128000, probs="f32", draft=True,
             shape=6),
        # One prompt continued eight times, every layer of the TinyLlama shape.
        dict(name="fork-samples", op="fork", n=1, forks=8, len_lo=713, len_hi=713, layers=22, kv=4, dim=64, cache="f16",
             page=16, shape=7),
        # A batch's prompts each continued twice more, every layer of the Llama-3 shape.
        dict(name="fork-batch", op="fork", n=24, forks=48, len_lo=100, len_hi=900, layers=32, kv=8, dim=128,
             cache="bf16", page=64, shape=8),
        # A few of a small batch's requests end.
        dict(name="free-few", op="free", n=16, len_lo=100, len_hi=4000, page=64, shape=9),
        # Half of a large batch over a large pool ends or is rolled back.
        dict(name="free-many", op="free", n=512, len_lo=0, len_hi=8000, page=16, shape=10),
        # A small pool after its requests came and went.
        dict(name="compact-few", op="compact", n=6, len_lo=20, len_hi=300, fill=50, layers=22, kv=4, dim=64,
             cache="f16", page=16, shape=11),
        # A large pool at half its use.
        dict(name="compact-batch", op="compact", n=32, len_lo=100, len_hi=1500, fill=55, layers=32, kv=8, dim=128,
             cache="bf16", page=64, shape=12),
    ]


HEADS = [(8, 2, 64), (12, 4, 64), (32, 4, 64), (20, 4, 128), (16, 16, 128), (32, 8, 128), (64, 8, 128)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "chunk", "verify", "verify", "fork", "free", "compact"])
    shape, page = rng.randrange(1, 1 << 30), rng.choice([16, 32, 64, 128])
    if op == "chunk":
        heads, kv, dim = rng.choice(HEADS)
        q, cache = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f16"), ("f32", "f32"),
                               ("f32", "bf16"), ("f32", "f16")])
        n = _log(rng, 1, 24)
        new = _log(rng, 1, 2500)
        # the padded scores of the plain form stay below the largest listed case's
        most = (30720 * 2048 * 32 if q != "f32" else 3000 * 1000 * 32) // (n * new * heads)
        if most < 2 * new:
            new = max(1, int((most * new / 2) ** 0.5))
            most = 2 * new
        len_hi = _log(rng, 1, max(1, min(30000, most - new)))
        return dict(op=op, n=n, len_lo=rng.choice([0, len_hi // 2, len_hi]), len_hi=len_hi,
                    new_lo=rng.choice([1, 0, new, -new]), new_hi=new, heads=heads, kv=kv, dim=dim, q=q, cache=cache,
                    page=page, shape=shape)
    if op == "verify":
        new, vocab = _log(rng, 1, 64), _log(rng, 300, 130000)
        n = _log(rng, 1, max(1, min(64, 48 * 17 * 128000 // (new * vocab))))
        return dict(op=op, n=n, new_lo=rng.choice([1, new]), new_hi=new, vocab=vocab,
                    probs=rng.choice(["f32", "f32", "f16", "bf16"]), draft=rng.random() < 0.6, shape=shape)
    if op == "free":
        return dict(op=op, n=_log(rng, 1, 500), len_lo=0, len_hi=_log(rng, 16, 8000), page=page, shape=shape)
    _, kv, dim = rng.choice(HEADS)
    layers, cache = _log(rng, 1, 32), rng.choice(["f32", "bf16", "f16"])
    if op == "fork":
        n = _log(rng, 1, 20)
        return dict(op=op, n=n, forks=_log(rng, 1, 2 * n + 6), len_lo=0, len_hi=_log(rng, 16, 800), layers=layers,
                    kv=min(kv, 8), dim=dim, cache=cache, page=page, shape=shape)
    return dict(op=op, n=_log(rng, 1, 20), len_lo=0, len_hi=_log(rng, 16, 800), fill=rng.choice([20, 50, 80, 100]),
                layers=min(layers, 16), kv=min(kv, 8), dim=dim, cache=cache, page=page, shape=shape)


def _sizes(case):
    """The ragged sizes of a case, the same for every seed."""
    r = random.Random(case["shape"])
    lens = [r.randint(case.get("len_lo", 0), case.get("len_hi", 0)) for _ in range(case["n"])]
    if case["op"] in ("chunk", "verify"):  # new_lo < 0: three quarters of the requests decode one token
        new = [r.randint(max(1, case["new_lo"]) if case["new_lo"] else 0, case["new_hi"]) for _ in range(case["n"])]
        if case["new_lo"] < 0:
            new = [1 if i % 4 else max(1, b) for i, b in enumerate(new)]
        new[0] = new[0] or case["new_hi"]
        return lens, new
    if case["op"] == "fork":
        return lens, [r.randrange(case["n"]) for _ in range(case["forks"])]
    if case["op"] == "free":  # requests end, are rolled back (refused where that ends inside a shared page), or stay
        return lens, [r.choice([0, 0, a // 2 // case["page"] * case["page"], a // 3, -1, -1]) for a in lens]
    pages = sum(-(-a // case["page"]) for a in lens)
    pool = max(pages, pages * 100 // case["fill"]) + 1
    return lens, r.sample(range(pool), pool)


def work(case):
    op = case["op"]
    lens, new = _sizes(case)
    if op == "verify":
        rows = sum(t > 0 for t in new) * (2 if case["draft"] else 1)
        return {"bytes": rows * case["vocab"] * SIZE[case["probs"]] + 24 * sum(new) + 16 * len(new), "flops": 0}
    ps = case["page"]
    if op == "chunk":
        row, h = case["kv"] * case["dim"], case["heads"] * case["dim"]
        return {"bytes": sum(2 * row * SIZE[case["cache"]] * (a + b) + 4 * -(-(a + b) // ps) for a, b in zip(lens, new) if b)
                + sum(new) * 2 * h * SIZE[case["q"]] + 8 * len(lens),
                "flops": sum(4 * h * (a * b + b * (b + 1) // 2) for a, b in zip(lens, new))}
    held = [-(-a // ps) for a in lens]
    if op == "free":
        pool = sum(held) + 5
        return {"bytes": 4 * (sum(h - -(-k // ps) for h, k in zip(held, new) if k >= 0) + 4 * pool + 6 * len(lens)),
                "flops": 0}
    row = case["layers"] * 2 * case["kv"] * case["dim"] * SIZE[case["cache"]]
    if op == "fork":
        return {"bytes": sum(2 * row * (lens[i] % ps) + 8 * held[i] for i in new) + 24 * len(new), "flops": 0}
    movers = sum(p >= sum(held) for p in new[:sum(held)])
    return {"bytes": 2 * row * ps * movers + 8 * sum(held) + 8 * len(new), "flops": 0}


# ---------------------------------------------------------------------------
# What a user's program holds
# ---------------------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(new):
    out = [0]
    for b in new:
        out.append(out[-1] + b)
    return out


def _tables(held, pages):
    """Block tables: the requests' pages one after another from `pages`."""
    table = torch.full((len(held), max(1, max(held)) + 1), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(held):
        table[i, :k] = pages[at:at + k]
        at += k
    return table.cuda()


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gc = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    lens, new = _sizes(case)
    if case["op"] == "verify":
        return _prepare_verify(s, new, g, gc)
    ps = case["page"]
    s["lens"] = _ints(lens)

    def normal(shape, dt):
        x = torch.empty(shape, device="cuda", dtype=DT[dt])
        return x.normal_(generator=gc)

    if case["op"] == "chunk":
        kv, d = case["kv"], case["dim"]
        need = [-(-(a + b) // ps) for a, b in zip(lens, new)]
        n_pages = sum(need) + 3
        s["table"] = _tables(need, torch.randperm(n_pages, generator=g).to(torch.int32))
        s["k_pool"], s["v_pool"] = (normal((n_pages, ps, kv, d), case["cache"]) for _ in "kv")
        s["q"] = normal((sum(new), case["heads"], d), case["q"])
        s["kv_lens"], s["node_start"] = _ints([a + b for a, b in zip(lens, new)]), _ints(_starts(new))
        return s
    held = [-(-a // ps) for a in lens]
    total = sum(held)
    if case["op"] == "free":
        # every fourth request shares its first full pages with the one before it
        n_pages = total + 5
        order = torch.randperm(n_pages, generator=g).to(torch.int32)
        table, shared, at = torch.full((len(lens), max(1, max(held)) + 1), -1, dtype=torch.int32), torch.zeros(n_pages), 0
        for i, k in enumerate(held):
            both = min(lens[i] // ps, lens[i - 1] // ps) // 2 if i % 4 == 3 else 0
            table[i, :both] = table[i - 1, :both]
            shared[table[i, :both].long()] += 1
            table[i, both:k] = order[at:at + k - both]
            at += k - both
        s["table"], s["shared"], s["free"] = table.cuda(), shared.int().cuda(), order.cuda()
        s["used"], s["owned"], s["keep"] = _ints([at]), _ints(held), _ints(new)
        return s
    layers, kv, d = case["layers"], case["kv"], case["dim"]
    if case["op"] == "fork":
        f = case["forks"]
        n_pages = total + f + 5
        order = torch.randperm(n_pages, generator=g).to(torch.int32)
        s["table"] = torch.cat((_tables(held, order), torch.full((f, max(1, max(held)) + 1), -1, dtype=torch.int32,
                                                                 device="cuda")))
        s["lens"], s["owned"] = _ints(lens + [0] * f), _ints(held + [0] * f)
        s["src"], s["dst"] = _ints(new), _ints(range(len(lens), len(lens) + f))
        s["free"], s["used"] = order.cuda(), _ints([total])
    else:
        n_pages = len(new)
        s["table"], s["owned"] = _tables(held, torch.tensor(new, dtype=torch.int32)), _ints(held)
    s["shared"] = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    s["k_pool"], s["v_pool"] = (normal((layers, n_pages, ps, kv, d), case["cache"]) for _ in "kv")
    return s


def _prepare_verify(s, new, g, gc):
    case = s["case"]
    total, vocab = sum(new), case["vocab"]
    parents, rank = [], []
    for t in new:  # the pending token, and drafts below it: most below a recent one
        below = [0] * t
        for j in range(t):
            a = max(0, j - 1 - int(torch.rand((), generator=g) ** 2 * 4)) if j else -1
            parents.append(a)
            rank.append(below[a] if j else 0)
            below[a] += 1 if j else 0
    start = _starts(new)
    first = torch.repeat_interleave(torch.tensor(start[:-1]), torch.tensor(new))
    above = (first + torch.tensor(parents).clamp(min=0)).cuda()
    # peaked distributions; the draft model's are the target's with some noise
    logits = torch.randn(total, vocab, generator=gc, device="cuda") * 3
    noisy = logits + torch.randn(total, vocab, generator=gc, device="cuda")
    s["target"] = torch.softmax(logits, -1).to(DT[case["probs"]])
    del logits
    if case["draft"]:
        noisy = torch.softmax(noisy, -1)
        s["draft"] = noisy.to(DT[case["probs"]])
        drawn = torch.rand(total, generator=gc, device="cuda")
        c = noisy.cumsum_(-1)
        tok = (c[above] < drawn[:, None] * c[above, -1:]).sum(-1).clamp(max=vocab - 1)
    else:
        s["draft"] = None
        tok = noisy.topk(min(8, vocab), -1).indices[above, torch.tensor(rank).clamp(max=7).cuda()]
    s["tokens"], s["parents"], s["node_start"] = tok.int(), _ints(parents), _ints(start)
    s["u"] = torch.rand(total, generator=gc, device="cuda")
    s["u_next"] = torch.rand(len(new), generator=gc, device="cuda")
    s["most"] = max(1, max(new))
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        import bml_b200
        if case["op"] == "chunk":
            return bml_b200.chunk_attention(s["q"], s["k_pool"], s["v_pool"], s["table"], s["kv_lens"], s["node_start"])
        if case["op"] == "verify":
            return bml_b200.verify_drafts(s["target"], s["draft"], s["tokens"], s["parents"], s["node_start"], s["u"],
                                          s["u_next"], max_path=s["most"])
        if case["op"] == "fork":
            p = bml_b200.page_fork(s["k_pool"], s["v_pool"], s["src"], s["dst"], s["lens"], s["owned"], s["table"],
                                   s["shared"], s["free"], s["used"])
            return p.lens, p.owned, p.shared, p.free_used, p.status, s["table"], s["k_pool"], s["v_pool"]
        if case["op"] == "free":
            p = bml_b200.page_free(s["keep"], s["lens"], s["owned"], s["table"], case["page"], s["shared"], s["free"],
                                   s["used"])
            return p.lens, p.owned, p.shared, p.free_pages, p.free_used, p.status
        p = bml_b200.page_compact(s["k_pool"], s["v_pool"], s["owned"], s["table"], s["shared"])
        return p.block_table, p.shared, p.free_pages, p.free_used, s["k_pool"], s["v_pool"]
    return {"chunk": _chunk, "verify": _verify, "fork": _fork, "free": _free, "compact": _compact}[case["op"]](s)


def _chunk(s):
    q, start, total = s["q"], s["node_start"].long(), s["kv_lens"].long()
    ps, kv, d = s["k_pool"].shape[1:]
    t_max = max(1, _sizes(s["case"])[1] and max(_sizes(s["case"])[1]))
    heads, group = q.shape[1], q.shape[1] // kv
    nodes = start[1:] - start[:-1]
    pos = torch.arange(s["table"].shape[1] * ps, device=q.device)
    rows = (s["table"].long()[:, pos // ps] * ps + pos % ps).clamp(min=0)
    k = s["k_pool"].reshape(-1, kv, d)[rows].float()              # [n, L, kv, d]
    v = s["v_pool"].reshape(-1, kv, d)[rows].float()
    t = torch.arange(t_max, device=q.device)
    out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    if q.shape[0] == 0:
        return out.to(q.dtype)
    tok = (start[:-1, None] + t).clamp(max=q.shape[0] - 1)        # [n, T]
    here = t < nodes[:, None]
    qs = q.float()[tok].reshape(len(total), t_max, kv, group, d)
    seen = pos <= (total - nodes)[:, None, None] + t[:, None]     # [n, T, L]
    sc = torch.einsum("ntkgd,nlkd->nkgtl", qs, k).mul_(1.0 / d ** 0.5)
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    l = sc.sum(-1)                                                # [n, kv, group, T]
    o = torch.einsum("nkgtl,nlkd->ntkgd", sc, v) / l.permute(0, 3, 1, 2)[..., None]
    out[tok[here]] = o.reshape(len(total), t_max, heads, d)[here]
    return out.to(q.dtype)


def _verify(s):
    p, draft, u = s["target"], s["draft"], s["u"].double()
    dev, start = p.device, s["node_start"].long()
    n, most, vocab = len(start) - 1, s["most"], p.shape[1]
    nodes = start[1:] - start[:-1]
    t = torch.arange(most, device=dev)
    here = t < nodes[:, None]                                     # [n, T]
    row = (start[:-1, None] + t).clamp(max=p.shape[0] - 1)
    tok = s["tokens"].long()[row]
    par = torch.where(here, s["parents"].long()[row], torch.full_like(row, -1))
    par = torch.where(par < t, par, torch.full_like(par, -1))
    same = (par[:, :, None] == par[:, None, :]) & (par >= 0)[:, :, None] & (t[:, None] > t)  # [n, T, T] an earlier sibling
    rank = same.sum(-1)
    again = (same & (tok[:, :, None] == tok[:, None, :])).any(-1)
    up = (start[:-1, None] + par.clamp(min=0)).clamp(max=p.shape[0] - 1)
    pv = p[up, tok].double()
    qv = draft[up, tok].double() if draft is not None else torch.ones_like(pv)
    uu = u[row]
    c, mass = (torch.full((n, most), x, dtype=torch.float64, device=dev) for x in (0.0, 1.0))
    chosen = torch.full((n, most), -1, device=dev)
    for k in range(int(rank.max()) + 1):  # the k-th child of every node
        kid = (par[:, None, :] == t[:, None]) & (rank == k)[:, None, :]        # [n, T, child]
        j = kid.long().argmax(-1)
        if draft is not None:
            r = (pv.gather(1, j) - c * qv.gather(1, j)).clamp(min=0)
        else:
            r = torch.where(again.gather(1, j), torch.zeros_like(pv), pv.gather(1, j))
        tried = kid.any(-1) & (chosen < 0)
        yes = tried & (uu.gather(1, j) * qv.gather(1, j) * mass < r)
        chosen = torch.where(yes, j, chosen)
        no = tried & ~yes
        if draft is not None:
            c = torch.where(no, c + mass, c)
            i, a = no.nonzero(as_tuple=True)
            at = start[i] + a
            mass[i, a] = (p[at].double() - c[i, a][:, None] * draft[at].double()).clamp_(min=0).sum(-1)
        else:
            mass = torch.where(no, mass - r, mass)
    # kept: every ancestor is its parent's chosen child
    good = (t == 0) | ((par >= 0) & (chosen.gather(1, par.clamp(min=0)) == t))
    see = (par[:, :, None] == t).double() + torch.eye(most, dtype=torch.float64, device=dev)
    see = torch.linalg.matrix_power(see, most) > 0                # [n, T, T] ancestors and itself
    kept = (~see | good[:, None, :]).all(-1) & see[:, :, 0] & here
    count = kept.sum(-1)
    path = torch.where(kept, t, torch.full_like(row, most)).sort(-1).values
    end = path.gather(1, (count - 1).clamp(min=0)[:, None])[:, 0].clamp(max=most - 1)
    at = (start[:-1] + end).clamp(max=p.shape[0] - 1)
    w = p[at].double()
    if draft is not None:
        w.addcmul_(draft[at].double(), c.gather(1, end[:, None]), value=-1.0)
    else:
        i, j = (par == end[:, None]).nonzero(as_tuple=True)
        w[i, tok[i, j]] = 0.0
    w.clamp_(min=0)
    cum = w.cumsum(-1)
    nxt = torch.searchsorted(cum, s["u_next"].double()[:, None] * cum[:, -1:], right=True)[:, 0].clamp(max=vocab - 1)
    nxt = torch.where(nodes > 0, nxt, torch.full_like(nxt, -1))
    path = torch.where(t < count[:, None], path, torch.full_like(path, -1))
    return path.int(), count.int(), nxt.int()


def _fork(s):
    ps = s["k_pool"].shape[2]
    src, dst, lens, table = s["src"].long(), s["dst"].long(), s["lens"].long(), s["table"]
    full, rest = lens[src] // ps, lens[src] % ps
    part = (rest > 0).long()
    fresh = s["free"].long()[(s["used"] + part.cumsum(0) - part).clamp(max=s["free"].numel() - 1)]
    j = torch.arange(table.shape[1], device=table.device)
    whole, last = j < full[:, None], (j == full[:, None]) & (part > 0)[:, None]
    rows = table[src]
    table[dst] = torch.where(whole, rows, torch.where(last, fresh.int()[:, None], table[dst]))
    shared = s["shared"].clone()
    shared.index_add_(0, rows.long().clamp(min=0).flatten(), whole.int().flatten())
    old = rows.long().gather(1, full[:, None].clamp(max=table.shape[1] - 1))[:, 0]
    i, r = (torch.arange(ps, device=table.device) < rest[:, None]).nonzero(as_tuple=True)
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, fresh[i], r] = pool[:, old[i], r]
    new_lens, owned = s["lens"].clone(), s["owned"].clone()
    new_lens[dst], owned[dst] = s["lens"][src], (full + part).int()
    return (new_lens, owned, shared, (s["used"] + part.sum()).int(), torch.zeros_like(s["src"]), table, s["k_pool"],
            s["v_pool"])


def _free(s):
    ps, table, free = s["case"]["page"], s["table"], s["free"].long()
    keep, lens, owned = s["keep"].long(), s["lens"].long(), s["owned"].long()
    new = torch.where(keep < 0, lens, torch.minimum(lens, keep))
    held = table.long().clamp(min=0)
    inside = held.gather(1, (new // ps).clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    refused = (new < lens) & (new % ps > 0) & (s["shared"][inside] > 0)
    new = torch.where(refused, lens, new)
    stay = torch.where((keep < 0) | refused, owned, torch.minimum(owned, (new + ps - 1) // ps))
    j = torch.arange(table.shape[1], device=table.device)
    drop = (j >= stay[:, None]) & (j < owned[:, None]) & (table >= 0)
    count = torch.zeros_like(s["shared"]).index_add_(0, held.flatten(), drop.int().flatten())
    gone = count > s["shared"]
    taken = torch.arange(len(free), device=free.device) < s["used"]
    key = torch.where(taken, gone[free].long(), torch.full_like(free, 2))
    order = free[torch.sort(key, stable=True).indices]
    return (new.int(), stay.int(), torch.where(gone, torch.zeros_like(count), s["shared"] - count), order.int(),
            (s["used"] - (key == 1).sum()).int(), refused.int() * 8)


def _compact(s):
    table, n_pages = s["table"], s["shared"].numel()
    dev = table.device
    live = torch.arange(table.shape[1], device=dev) < s["owned"][:, None]
    mark = torch.zeros(n_pages, dtype=torch.int32, device=dev)
    mark.index_add_(0, table.long().clamp(min=0).flatten(), live.int().flatten())
    page = torch.arange(n_pages, device=dev)
    used = (mark > 0).sum()
    mover, hole = ((mark > 0) & (page >= used)).nonzero()[:, 0], ((mark == 0) & (page < used)).nonzero()[:, 0]
    to = page.clone()
    to[mover] = hole
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, hole] = pool[:, mover]
    shared = torch.zeros_like(s["shared"])
    shared[to[mark > 0]] = s["shared"][mark > 0]
    return (torch.where(live, to[table.long().clamp(min=0)].int(), table), shared, page.int(), used.int()[None],
            s["k_pool"], s["v_pool"])


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] != "chunk":  # whole numbers, and rows that only move
        return None
    s = prepare(case, seed)
    lens, new = _sizes(case)
    group, out, at = case["heads"] // case["kv"], [], 0
    for i, (a, b) in enumerate(zip(lens, new)):
        if b == 0:
            continue
        pages = s["table"][i, :-(-(a + b) // case["page"])].long()
        late = torch.arange(a + b, device="cuda") > a + torch.arange(b, device="cuda")[:, None]
        heads = []
        for h in range(case["heads"]):
            k = s["k_pool"][pages, :, h // group].flatten(0, 1)[:a + b].double()
            v = s["v_pool"][pages, :, h // group].flatten(0, 1)[:a + b].double()
            x = (s["q"][at:at + b, h].double() @ k.T) / case["dim"] ** 0.5
            heads.append(torch.softmax(x.masked_fill_(late, float("-inf")), -1) @ v)
        out.append(torch.stack(heads, 1))
        at += b
    return torch.cat(out, 0) if out else torch.zeros(0, case["heads"], case["dim"], dtype=torch.float64, device="cuda")
