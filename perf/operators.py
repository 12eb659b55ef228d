"""The work that four operators of the paged cache are measured on: attention for trees of drafted tokens, the acceptance of a
tree with the move of its accepted rows, attention that adds up every cached row's weight, and the eviction of the rows that
gathered least.

A case is one call as a serving program makes it between two projections of a layer (the attentions) or once a step for all
layers (acceptance, eviction). The cache is the package's own: pages of 64 rows, [pages, kv heads, 64, head], a list of pages
for every sequence, in no particular order. With `own` false a pass is elementary torch arithmetic on the same tensors, in 32
bits and rounded once; with `own` true it is the package's call.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

PAGE = 64
VOCAB = 151936

TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# -------------------------------------------------------------------- cases

def _tree(name, batch, rows, past, heads, kv, dim, dtype="bfloat16"):
    c = {"op": "tree", "batch": batch, "rows": rows, "past": past, "heads": heads, "kv": kv, "dim": dim, "dtype": dtype}
    return dict(c, name=name) if name else c


def _mass(name, batch, rows, past, heads, kv, dim, dtype="bfloat16"):
    c = {"op": "mass", "batch": batch, "rows": rows, "past": past, "heads": heads, "kv": kv, "dim": dim, "dtype": dtype}
    return dict(c, name=name) if name else c


def _evict(name, layers, batch, held, keep, recent, first, kv, dim, dtype="bfloat16"):
    c = {"op": "evict", "layers": layers, "batch": batch, "held": held, "keep": keep, "recent": recent, "first": first, "kv": kv,
         "dim": dim, "dtype": dtype}
    return dict(c, name=name) if name else c


def _commit(name, layers, batch, rows, past, kv, dim, dtype="bfloat16"):
    c = {"op": "commit", "layers": layers, "batch": batch, "rows": rows, "past": past, "kv": kv, "dim": dim, "dtype": dtype}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user, a few drafted tokens behind a short conversation: latency is what counts
        _tree("tree-1x8", 1, 8, 1000, 16, 8, 128),
        # a batch of conversations of unequal lengths, trees of two dozen tokens
        _tree("tree-8x24", 8, 24, 2050, 16, 8, 128),
        # a full server: large trees behind long contexts, four query heads on a kv head
        _tree("tree-16x64-long", 16, 64, 8191, 32, 8, 128),
        # the true 32-bit path with heads of 64
        _tree("tree-fp32", 3, 19, 1021, 12, 4, 64, "float32"),
        # a decode step of one sequence behind a bounded cache
        _mass("mass-decode-1", 1, 1, 1535, 16, 8, 128),
        # a decode step of many sequences of unequal lengths
        _mass("mass-decode-64", 64, 1, 4000, 32, 8, 128),
        # a whole prompt, whose rows start their sums
        _mass("mass-prompt", 1, 2048, 0, 16, 8, 128),
        # a further piece of two prompts, in 32 bits with heads that no tensor core takes
        _mass("mass-piece-fp32", 2, 150, 333, 6, 3, 48, "float32"),
        # one layer's cache of one sequence, a little over its bound
        _evict("evict-1", 1, 1, 700, 512, 64, 4, 8, 128),
        # all layers of two sequences that have filled twice what they keep
        _evict("evict-layers", 28, 2, 4100, 2048, 256, 16, 8, 128),
        # the step of one user: eight drafted tokens, all layers
        _commit("commit-1x8", 28, 1, 8, 1000, 8, 128),
        # the step of a server: large trees, all layers
        _commit("commit-32x64", 36, 32, 64, 1029, 8, 128),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["tree", "mass", "evict", "commit"])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    kv = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128, 128] if dtype == "bfloat16" else [48, 64, 128])
    while True:
        heads = kv * rng.choice([1, 2, 3, 4, 5, 8])
        if op == "tree":
            c = _tree(None, _log(rng, 1, 32), _log(rng, 1, 100), _log(rng, 1, 16000), heads, kv, dim, dtype)
        elif op == "mass":
            c = _mass(None, _log(rng, 1, 64), rng.choice([1, _log(rng, 2, 3000)]), _log(rng, 1, 8000) - 1, heads, kv, dim, dtype)
        elif op == "evict":
            held = _log(rng, 70, 16000)
            keep = max(2, int(held * rng.uniform(0.2, 0.95)))
            recent = rng.randint(0, keep // 2)
            c = _evict(None, _log(rng, 1, 28), _log(rng, 1, 4), held, keep, recent, rng.randint(0, min(16, keep - recent)), kv, dim, dtype)
        else:
            c = _commit(None, _log(rng, 1, 36), _log(rng, 1, 32), _log(rng, 1, 128), _log(rng, 1, 4000), kv, dim, dtype)
        # no dearer than the largest listed case: what a pass computes, what it moves and what its state holds
        w = work(c)
        limit = 8e10 if dtype == "bfloat16" else 8e9
        pools = c.get("layers", 1) * c["batch"] * (c.get("past", c.get("held", 0)) + c.get("rows", 0) + 128) * kv * dim * 8
        scores = c["batch"] * c.get("heads", 0) * c.get("rows", 0) * (c.get("past", 0) + c.get("rows", 0)) * 4 if op in ("tree", "mass") else 0
        if w["flops"] <= limit and w["bytes"] <= 9e8 and pools <= 8e9 and scores <= 1.2e9:
            return c


def _lengths(case):
    """Rows that every sequence holds before the step's own (for an eviction: all it holds): the longest as the case says, the
    others less."""
    top, batch = case["held"] if case["op"] == "evict" else case["past"], case["batch"]
    return [top - (b * 37) % max(1, top // 2 + 1) if b else top for b in range(batch)]


def _rows(case):
    """New rows of every sequence: the first as the case says, the others up to a third fewer."""
    return [case["rows"] - (b * 5) % max(1, case["rows"] // 3 + 1) for b in range(case["batch"])]


def work(case):
    es = 2 if case["dtype"] == "bfloat16" else 4
    kv, dim = case["kv"], case["dim"]
    if case["op"] in ("tree", "mass"):
        heads, past, rows = case["heads"], _lengths(case), _rows(case)
        kv_rows, q_rows = sum(past) + sum(rows), sum(rows)
        byts = kv_rows * kv * dim * 2 * es + q_rows * heads * dim * 2 * es
        if case["op"] == "tree":      # a row sees what was held and, at the least, itself
            pairs = sum(n * (p + 1) for p, n in zip(past, rows))
            byts += q_rows * 8 * (-(-case["rows"] // 64))
        else:                         # causal; the sums of the held rows are read, all are written
            pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, rows))
            byts += (sum(past) + kv_rows) * kv * 4
        return {"bytes": byts, "flops": 4 * pairs * heads * dim}
    layers = case["layers"]
    if case["op"] == "evict":
        held = _lengths(case)
        kept = sum(min(n, case["keep"]) for n in held)
        # all sums are read; what is kept is read and written; the choice is written
        byts = layers * kv * (sum(held) * 4 + kept * (2 * (2 * dim * es) + 4) + kept * 4)
        return {"bytes": byts, "flops": layers * kv * sum(held)}
    rows = _rows(case)
    moved = sum(max(1, n // 4) for n in rows)                       # about the rows that a path of the tree has
    return {"bytes": layers * kv * moved * 2 * (2 * dim * es) + sum(rows) * 16, "flops": sum(rows)}


# ------------------------------------------------------------------- states

def _pages(lens, gen, spare=0):
    """Page lists in no order: (indptr, ids, base, pages of the pool, the lists as a padded table)."""
    counts = [-(-n // PAGE) for n in lens]
    total = sum(counts) + spare
    ids = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    most = max(max(counts), 1)
    at = torch.tensor(starts[:-1], device="cuda")[:, None] + torch.arange(most, device="cuda")[None, :]
    table = ids[at.clamp(max=max(total - 1, 0))].to(torch.int64)     # entries behind a sequence's last page are never used
    return SimpleNamespace(indptr=torch.tensor(starts, dtype=torch.int32, device="cuda"), ids=ids[:starts[-1]].contiguous(),
                           base=torch.zeros(len(lens), dtype=torch.int32, device="cuda"), n_pages=total), table, ids[starts[-1]:]


def _randn(shape, dtype, gen):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _forest(rows, width, gen):
    """Trees: every row but a sequence's first hangs on an earlier one, most on one of the last few. Returns parents [T] and the
    rows' ancestors and selves as words of 64 bits [T, words]."""
    parents, masks = [], []
    for n in rows:
        i = torch.arange(n, device="cuda")
        back = (torch.rand(n, generator=gen, device="cuda").pow(2) * torch.clamp(i, max=8)).long() + 1
        p = torch.where(i > 0, torch.clamp(i - back, min=0), -1)
        hang = torch.zeros((n, n), dtype=torch.float64, device="cuda")
        if n > 1:
            hang[i[1:], p[1:]] = 1.0
        seen = torch.linalg.solve_triangular(torch.eye(n, dtype=torch.float64, device="cuda") - hang,
                                             torch.eye(n, dtype=torch.float64, device="cuda"), upper=False)
        bits = torch.zeros((n, width * 64), dtype=torch.int64, device="cuda")
        bits[:, :n] = (seen > 0.5).long()
        words = (bits.view(n, width, 64) << torch.arange(64, device="cuda")).sum(-1)
        parents.append(p.to(torch.int32))
        masks.append(words)
    return torch.cat(parents), torch.cat(masks)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype, kv, dim, batch = TYPES[case["dtype"]], case["kv"], case["dim"], case["batch"]
    past = _lengths(case)
    rows = [0] * batch if case["op"] == "evict" else _rows(case)
    held = [p + n for p, n in zip(past, rows)]
    pages, table, spare = _pages(held, gen, spare=batch * -(-case["keep"] // PAGE) if case["op"] == "evict" else 2)
    cu = [0]
    for n in rows:
        cu.append(cu[-1] + n)
    ctx = SimpleNamespace(B=batch, T=cu[-1], max_q_len=max(rows), cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"),
                          kv_len=torch.tensor(held, dtype=torch.int32, device="cuda"), pages=[pages],
                          status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    s = SimpleNamespace(case=case, ctx=ctx, pages=pages, table=table, kv=kv, dim=dim)
    if case["op"] in ("tree", "mass"):
        heads = case["heads"]
        # keys of unit size, a few of which all queries look for (the rows that gather weight); values behind them
        to = _randn((kv, 1, dim), torch.float32, gen)
        k = _randn((pages.n_pages, kv, PAGE, dim), torch.float32, gen)
        k += to * 0.8 * (torch.rand((pages.n_pages, kv, PAGE, 1), generator=gen, device="cuda") < 0.05)
        s.k, s.v = k.to(dtype), _randn((pages.n_pages, kv, PAGE, dim), dtype, gen)
        q = _randn((cu[-1], kv, heads // kv, dim), torch.float32, gen) + 0.3 * to
        s.q = q.to(dtype).view(cu[-1], heads * dim)
        s.out = torch.zeros((cu[-1], heads * dim), dtype=dtype, device="cuda")
        s.heads, s.scale = heads, dim ** -0.5
        if case["op"] == "tree":
            s.parents, s.masks = _forest(rows, -(-max(rows) // 64), gen)
        else:
            s.mass = torch.rand((pages.n_pages, kv, PAGE), generator=gen, device="cuda") ** 8 * 4.0
        return s
    layers = case["layers"]
    s.k = _randn((layers, pages.n_pages, kv, PAGE, dim), dtype, gen)
    s.v = _randn((layers, pages.n_pages, kv, PAGE, dim), dtype, gen)
    if case["op"] == "evict":
        # weights that a row has gathered: a few rows have most of it, many next to nothing, some exactly nothing
        m = torch.rand((layers, pages.n_pages, kv, PAGE), generator=gen, device="cuda") ** 12 * 50.0
        s.mass = torch.where(m < 1e-6, torch.zeros_like(m), m)
        each = -(-case["keep"] // PAGE)
        s.to = SimpleNamespace(indptr=torch.arange(0, (batch + 1) * each, each, dtype=torch.int32, device="cuda"),
                               ids=spare.contiguous(), base=pages.base, n_pages=pages.n_pages)
        s.to_table = spare.view(batch, each).to(torch.int64)
        return s
    s.parents, s.masks = _forest(rows, -(-max(rows) // 64), gen)
    n = cu[-1]
    s.tokens = torch.randint(0, VOCAB, (n,), generator=gen, device="cuda", dtype=torch.int32)
    # what the model would say behind every row: one of its children's tokens more often than not
    s.chosen = torch.randint(0, VOCAB, (n,), generator=gen, device="cuda", dtype=torch.int32)
    first = torch.repeat_interleave(ctx.cu_q[:-1].long(), torch.tensor(rows, device="cuda"))
    has = (s.parents >= 0) & (torch.rand(n, generator=gen, device="cuda") < 0.9)
    at = torch.where(has, first + s.parents.long(), n)
    # of several children the last one's token: a maximum, so that the order of writes does not matter
    best = torch.full((n + 1,), -1, dtype=torch.int64, device="cuda").scatter_reduce(0, at, torch.arange(n, device="cuda"), "amax")[:n]
    s.chosen = torch.where(best >= 0, s.tokens[best.clamp(min=0)], s.chosen)
    return s


# -------------------------------------------------------------- plain forms

def _plain_attention(s):
    """Both attentions: every sequence padded to the longest, all scores at once. Returns the outputs and the weights
    [batch, kv, group, rows, held]."""
    c, kv, dim = s.ctx, s.kv, s.dim
    group = s.heads // kv
    n, most = c.max_q_len, s.table.shape[1] * PAGE
    k = s.k[s.table].permute(0, 2, 1, 3, 4).reshape(c.B, kv, most, dim).float()
    v = s.v[s.table].permute(0, 2, 1, 3, 4).reshape(c.B, kv, most, dim).float()
    cu, held = c.cu_q.long(), c.kv_len.long()
    rows = cu[1:] - cu[:-1]
    past = held - rows
    i = torch.arange(n, device=s.q.device)
    at = (cu[:-1, None] + i).clamp(max=s.q.shape[0] - 1)
    there = i[None, :] < rows[:, None]
    q = s.q[at].float().view(c.B, n, kv, group, dim).permute(0, 2, 3, 1, 4)
    r = torch.arange(most, device=s.q.device)
    if s.case["op"] == "tree":
        j = r[None, :] - past[:, None]
        word = s.masks[at].gather(2, (j.clamp(min=0) // 64).clamp(max=s.masks.shape[1] - 1)[:, None, :].expand(c.B, n, most))
        sees = (j[:, None, :] < 0) | (((word >> (j.clamp(min=0) % 64)[:, None, :]) & 1) == 1)
    else:
        sees = r[None, None, :] <= past[:, None, None] + i[None, :, None]
    sees = sees & (r[None, None, :] < held[:, None, None]) & there[:, :, None]
    v = torch.where((r[None, :] < held[:, None])[:, None, :, None], v, 0.0)
    w = torch.matmul(q.reshape(c.B, kv, group * n, dim), k.transpose(2, 3)).view(c.B, kv, group, n, most)
    w = (w * s.scale).masked_fill_(~sees[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(torch.isinf(top), 0.0, top))
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-38)
    out = torch.matmul(w.view(c.B, kv, group * n, most), v).view(c.B, kv, group, n, dim).permute(0, 3, 1, 2, 4).reshape(c.B, n, -1)
    # rows of a sequence stand one behind the other again: T rows, each from its place in the padded block
    b = torch.repeat_interleave(torch.arange(c.B, device=s.q.device), rows, output_size=c.T)
    return out[b, torch.arange(c.T, device=s.q.device) - cu[b]].to(s.q.dtype), w, past, held


def _plain_tree(s):
    out, _, _, _ = _plain_attention(s)
    return {"out": out}


def _plain_mass(s):
    out, w, past, held = _plain_attention(s)
    most = s.table.shape[1] * PAGE
    new = w.sum((2, 3))                                                          # [batch, kv, held]
    r = torch.arange(most, device=s.q.device)
    old = s.mass[s.table].permute(0, 2, 1, 3).reshape(s.ctx.B, s.kv, most)
    new = new + torch.where((r[None, :] < past[:, None])[:, None, :], old, 0.0)
    new = torch.where((r[None, :] < held[:, None])[:, None, :], new, old)       # rows behind the last stay as they are
    ok = torch.arange(s.table.shape[1], device=s.q.device)[None, :] * PAGE < held[:, None]
    full = new.view(s.ctx.B, s.kv, -1, PAGE).permute(0, 2, 1, 3)
    # a padded table names pages of other sequences behind a sequence's last: those are not written
    dst = torch.where(ok, s.table, s.mass.shape[0])
    s.mass = torch.cat([s.mass, s.mass[:1]]).index_copy(0, dst.reshape(-1), full.reshape(-1, s.kv, PAGE))[:-1]
    return {"out": out, "mass": s.mass}


def _plain_evict(s):
    c, kv, keep = s.ctx, s.kv, s.case["keep"]
    first, recent = s.case["first"], s.case["recent"]
    layers = s.k.shape[0]
    most = s.table.shape[1] * PAGE
    held = c.kv_len.long()
    r = torch.arange(most, device=s.k.device)
    m = s.mass[:, s.table].permute(0, 1, 3, 2, 4).reshape(layers, c.B, kv, most)
    must = (r[None, :] < first) | (r[None, :] >= held[:, None] - recent)
    rank = torch.where(must[None, :, None, :], math.inf, m)
    rank = torch.where((r[None, :] < held[:, None])[None, :, None, :], rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    n = held.clamp(max=keep)
    i = torch.arange(keep, device=s.k.device)
    there = (i[None, :] < n[:, None])[None, :, None, :]
    kept = torch.where(there, order, most).sort(-1).values
    kept = torch.where(there, kept, -1)
    src = kept.clamp(min=0)
    e = torch.arange(layers, device=s.k.device)[:, None, None, None]
    b = torch.arange(c.B, device=s.k.device)[None, :, None, None]
    g = torch.arange(kv, device=s.k.device)[None, None, :, None]
    sp, sr = s.table[b, src // PAGE], src % PAGE
    dp, dr = s.to_table[b, (i // PAGE)[None, None, None, :]], (i % PAGE)[None, None, None, :]
    for t in (s.k, s.v):
        t[e, dp, g, dr] = torch.where(there[..., None], t[e, sp, g, sr], t[e, dp, g, dr])
    s.mass[e, dp, g, dr] = torch.where(there, s.mass[e, sp, g, sr], s.mass[e, dp, g, dr])
    return {"kept": kept.to(torch.int32), "kv_len": n.to(torch.int32), "k": s.k, "v": s.v, "mass": s.mass}


def _plain_commit(s):
    c, n = s.ctx, s.ctx.max_q_len
    cu, held = c.cu_q.long(), c.kv_len.long()
    rows = cu[1:] - cu[:-1]
    i = torch.arange(n, device=s.k.device)
    at = (cu[:-1, None] + i).clamp(max=c.T - 1)
    there = i[None, :] < rows[:, None]
    parent = torch.where(there, s.parents[at].long(), -1)
    token, chosen = s.tokens[at], s.chosen[at]
    hangs = parent.clamp(min=0)
    good = there & (parent >= 0) & (token == chosen.gather(1, hangs))
    twin = good[:, :, None] & good[:, None, :] & (parent[:, :, None] == parent[:, None, :])     # several good children of one row
    good = good & ~(twin & (i[None, None, :] < i[None, :, None])).any(-1)
    good = good | (there & (i == 0)[None, :])
    # ancestors: the inverse of (1 - parent matrix) has a one for every row above a row
    hang = ((parent[:, :, None] == i[None, None, :]) & there[:, :, None]).double()
    above = torch.linalg.solve_triangular(torch.eye(n, dtype=torch.float64, device=s.k.device) - hang,
                                          torch.eye(n, dtype=torch.float64, device=s.k.device).expand(c.B, n, n), upper=False) > 0.5
    on = there & ~(above & ~good[:, None, :]).any(-1) & above[:, :, 0]
    count = on.sum(-1)
    last = torch.where(on, i[None, :], -1).amax(-1)
    path = torch.where(on, i[None, :], n).sort(-1).values
    path = torch.where(i[None, :] < count[:, None], path, -1)
    after = torch.where(count > 0, chosen.gather(1, last.clamp(min=0)[:, None])[:, 0].long(), -1)
    # row i of a sequence's new rows takes row path[i], or stays; places behind a sequence's last repeat the last
    to = torch.minimum(i[None, :], (rows - 1)[:, None])
    off = torch.where(to < count[:, None], path.gather(1, to), to)
    src, dst = (held - rows)[:, None] + off, (held - rows)[:, None] + to
    b = torch.arange(c.B, device=s.k.device)[:, None]
    sp, sr, dp, dr = s.table[b, src // PAGE], src % PAGE, s.table[b, dst // PAGE], dst % PAGE
    for t in (s.k, s.v):
        t[:, dp, :, dr] = t[:, sp, :, sr]
    flat = torch.repeat_interleave(torch.arange(c.B, device=s.k.device), rows, output_size=c.T)
    path = path[flat, torch.arange(c.T, device=s.k.device) - cu[flat]]
    return {"path": path.to(torch.int32), "count": count.to(torch.int32), "next": after.to(torch.int32), "k": s.k, "v": s.v}


# ---------------------------------------------------------------------- run

def run(s):
    op = s.case["op"]
    if not own:
        return {"tree": _plain_tree, "mass": _plain_mass, "evict": _plain_evict, "commit": _plain_commit}[op](s)
    from mynah_slm_b200.ops import evict, tree
    if op == "tree":
        tree.attn_tree(s.q, s.out, s.ctx, s.heads, s.kv, s.dim, s.k, s.v, s.pages, s.masks, s.scale)
        return {"out": s.out}
    if op == "mass":
        evict.attn_mass(s.q, s.out, s.mass, s.ctx, s.heads, s.kv, s.dim, s.k, s.v, s.pages, s.scale)
        return {"out": s.out, "mass": s.mass}
    if op == "evict":
        kept, n = evict.cache_evict(s.k, s.v, s.mass, s.ctx, s.pages, s.case["keep"], s.case["recent"], s.case["first"], out_pages=s.to)
        return {"kept": kept, "kv_len": n, "k": s.k, "v": s.v, "mass": s.mass}
    path, count, after = tree.tree_commit(s.tokens, s.parents, s.chosen, s.ctx, s.k, s.v, s.pages)
    return {"path": path, "count": count, "next": after, "k": s.k, "v": s.v}


# -------------------------------------------------------------------- exact

def exact(case, seed):
    """From the definitions, sequence by sequence and row by row where that is the definition; sums in 64 bits."""
    s = prepare(case, seed)
    kv, dim = s.kv, s.dim
    past, rows = _lengths(case), _rows(case) if case["op"] != "evict" else None
    if case["op"] in ("tree", "mass"):
        heads = s.heads
        out = torch.zeros((s.ctx.T, heads, dim), dtype=torch.float64, device="cuda")
        mass = s.mass.double() if case["op"] == "mass" else None
        at = 0
        for b, (p, n) in enumerate(zip(past, rows)):
            held = p + n
            pages = s.table[b, :-(-held // PAGE)]
            sees = torch.ones((n, held), dtype=torch.bool, device="cuda")
            if case["op"] == "tree":
                for j in range(n):
                    sees[:, p + j] = (s.masks[at:at + n, j // 64] >> (j % 64)) & 1 == 1
            else:
                sees[:, p:] = torch.ones((n, n), device="cuda").tril() > 0
            for g in range(kv):
                k = s.k[pages, g].reshape(-1, dim)[:held].double()
                v = s.v[pages, g].reshape(-1, dim)[:held].double()
                total = torch.zeros(held, dtype=torch.float64, device="cuda")
                for h in range(g * (heads // kv), (g + 1) * (heads // kv)):
                    z = s.q[at:at + n, h * dim:(h + 1) * dim].double() @ k.T * s.scale
                    z = torch.softmax(torch.where(sees, z, -torch.inf), -1)
                    out[at:at + n, h] = z @ v
                    total += z.sum(0)
                if mass is not None:
                    total[:p] += s.mass[pages, g].reshape(-1)[:p].double()
                    last = s.mass[pages, g].reshape(-1).double()
                    last[:held] = total
                    mass[pages, g] = last.view(-1, PAGE)
            at += n
        out = out.view(s.ctx.T, heads * dim)
        return {"out": out} if mass is None else {"out": out, "mass": mass}
    if case["op"] == "evict":
        if case["layers"] * case["batch"] * kv > 1000:
            return None
        keep, recent, first = case["keep"], case["recent"], case["first"]
        kept = torch.full((case["layers"], case["batch"], kv, keep), -1, dtype=torch.int32)
        k2, v2, m2 = s.k.clone(), s.v.clone(), s.mass.clone()
        for b, n in enumerate(past):
            pages = s.table[b, :-(-n // PAGE)]
            to = s.to_table[b]
            for e in range(case["layers"]):
                sums = s.mass[e, pages].permute(1, 0, 2).reshape(kv, -1)[:, :n].cpu().double()
                for g in range(kv):
                    if n <= keep:
                        rows_kept = torch.arange(n)
                    else:
                        middle = sums[g, first:n - recent]
                        best = torch.argsort(-middle, stable=True)[:keep - first - recent] + first
                        rows_kept = torch.cat([torch.arange(first), best.sort().values, torch.arange(n - recent, n)])
                    kept[e, b, g, :rows_kept.numel()] = rows_kept.to(torch.int32)
                    src, dst = rows_kept.cuda(), torch.arange(rows_kept.numel(), device="cuda")
                    for x, y in ((s.k, k2), (s.v, v2), (s.mass, m2)):
                        y[e, to[dst // PAGE], g, dst % PAGE] = x[e, pages[src // PAGE], g, src % PAGE]
        n = torch.tensor([min(n, keep) for n in past], dtype=torch.int32)
        return {"kept": kept, "kv_len": n, "k": k2, "v": v2, "mass": m2}
    tokens, parents, chosen = s.tokens.tolist(), s.parents.tolist(), s.chosen.tolist()
    path, count, after = [], [], []
    k2, v2 = s.k.clone(), s.v.clone()
    at = 0
    for b, (p, n) in enumerate(zip(past, rows)):
        walk = [0]
        while True:
            nxt = [c for c in range(1, n) if parents[at + c] == walk[-1] and tokens[at + c] == chosen[at + walk[-1]]]
            if not nxt:
                break
            walk.append(nxt[0])
        path += walk + [-1] * (n - len(walk))
        count.append(len(walk))
        after.append(chosen[at + walk[-1]])
        src = torch.tensor(walk, device="cuda") + p
        dst = torch.arange(len(walk), device="cuda") + p
        for x, y in ((s.k, k2), (s.v, v2)):
            y[:, s.table[b, dst // PAGE], :, dst % PAGE] = x[:, s.table[b, src // PAGE], :, src % PAGE]
        at += n
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"path": i32(path), "count": i32(count), "next": i32(after), "k": k2, "v": v2}
