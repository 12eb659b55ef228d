"""Attention for trees of drafted tokens and the acceptance of a tree, against the definitions in 64 bits."""
import random

import numpy as np
import pytest
import torch

from plain import rows as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _tree(n, rng, roots=False):
    return [-1 if i == 0 or (roots and rng.random() < 0.1) else max(0, i - 1 - int(rng.random() ** 2 * 6)) for i in range(n)]


def _masks(trees, words=None):
    from mynah_slm_b200.ops.tree import tree_rows
    words = words or max(1, max(-(-len(t) // 64) for t in trees))
    parts = [torch.from_numpy(tree_rows(t, words)[1].copy()) for t in trees if t]
    return torch.cat(parts) if parts else torch.zeros((0, words), dtype=torch.int64)


def _case(seed, rows, past, H, KV, HD, dtype, pad=0, wide=0):
    g = _gen(seed)
    step = plain.make_step(rows, past, DEV, g)
    T = sum(rows) + pad
    q = torch.randn((T, H * HD + wide), generator=g).to(dtype)
    k = torch.randn((step.pages.n_pages, KV, 64, HD), generator=g).to(dtype)
    v = torch.randn((step.pages.n_pages, KV, 64, HD), generator=g).to(dtype)
    return step, q, k, v


def _tensor_cores(dtype, H, KV, HD):
    return dtype == BF16 and HD in (64, 128) and H // KV <= 128


def _check(step, q, k, v, H, KV, HD, masks, dtype, scale=0.0, got=None, pad=0):
    """Runs attn_tree and compares; returns the output."""
    from mynah_slm_b200.ops import tree
    T = sum(step.q_lens) + pad
    out = torch.full((T, H * HD), 7.0, dtype=dtype, device=DEV)
    qd = q.to(DEV)
    full = torch.zeros((T, masks.shape[1]), dtype=torch.int64)
    full[:masks.shape[0]] = masks
    tree.attn_tree(qd, out, step, H, KV, HD, k.to(DEV), v.to(DEV), step.pages, full.to(DEV), scale)
    torch.cuda.synchronize()
    assert step.status.item() == 0
    tc = _tensor_cores(dtype, H, KV, HD)
    ref, bound, _, _ = plain.attention(step, q[:, :H * HD], k, v, H, scale or HD ** -0.5, plain.by_words(step, masks),
                                       2.0 ** -8 if tc else 0.0, 2 * plain.F32 if tc else plain.F32)
    n = sum(step.q_lens)
    ref, bound = ref[:n], bound[:n]
    o = out[:n].double().cpu().view(n, H, HD)
    last = 2.0 ** -8 if dtype == BF16 else plain.F32
    tol = bound + last * (ref.abs() + bound) + 1e-37
    bad = ~((o - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values, worst {float(((o - ref).abs() / tol).nan_to_num(1e9).max()):.2f} of the bound"
    assert (out[n:] == 7.0).all(), "rows behind the last sequence"
    return out


CASES = [  # rows, past, H, KV, HD
    ([1], [0], 2, 1, 64), ([1], [1], 4, 2, 128), ([5], [63], 4, 2, 64), ([8], [64], 16, 8, 128), ([7], [65], 6, 2, 128),
    ([64], [0], 4, 2, 64), ([64, 1, 33], [130, 500, 63], 8, 2, 128), ([100], [200], 8, 1, 64), ([70, 130], [61, 1], 2, 2, 128),
    ([3, 0, 9, 0], [10, 0, 700, 40], 10, 2, 64), ([24] * 5, [300, 20, 64, 127, 128], 4, 4, 128), ([17], [3000], 16, 2, 128),
    ([20], [100], 12, 4, 48), ([6, 40], [77, 3], 5, 5, 8), ([9], [150], 6, 3, 80), ([33], [129], 4, 1, 256), ([4], [90], 40, 1, 64),
    ([2], [70], 200, 1, 64), ([65], [0], 3, 1, 128), ([128], [64], 5, 1, 64),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}-{c[2]}:{c[3]}x{c[4]}".replace(" ", ""))
def test_tree_attention_is_the_formula(case, dtype):
    rows, past, H, KV, HD = case
    rng = random.Random(len(rows) * 1000 + H)
    step, q, k, v = _case(7, rows, past, H, KV, HD, dtype)
    _check(step, q, k, v, H, KV, HD, _masks([_tree(n, rng) for n in rows]), dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_any_mask_rows_that_see_nothing_and_words_behind_the_rows(dtype):
    rows, past, H, KV, HD = [40, 70], [0, 0], 4, 2, 64
    step, q, k, v = _case(11, rows, past, H, KV, HD, dtype)
    g = _gen(3)
    masks = torch.randint(-2 ** 62, 2 ** 62, (sum(rows), 3), generator=g)      # bits behind the last row are set too
    masks[5] = 0
    masks[40:60] = 0
    masks[66, 1:] = 0
    masks[66, 0] = -2 ** 63                            # row 63 alone
    out = _check(step, q, k, v, H, KV, HD, masks, dtype)
    assert (out[5] == 0).all() and (out[40:60] == 0).all()
    # too few words: rows beyond them are seen by nobody
    _check(step, q, k, v, H, KV, HD, masks[:, :1].contiguous(), dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("HD", [64, 128, 48])
def test_what_lies_in_unseen_rows_has_no_influence(dtype, HD):
    rows, past, H, KV = [20, 70], [50, 130], 4, 2
    rng = random.Random(5)
    trees = [_tree(n, rng, roots=True) for n in rows]
    step, q, k, v = _case(13, rows, past, H, KV, HD, dtype)
    masks = _masks(trees)
    clean = _check(step, q, k, v, H, KV, HD, masks, dtype)
    # one drafted row of each sequence that some rows see and others do not, and every row behind the last
    seen = plain.by_words(step, masks)
    for fill in (float("nan"), float("inf"), float("-inf")):
        k2, v2 = k.clone(), v.clone()
        for b, row in ((0, 3), (1, 40)):
            at = past[b] + row
            for t in (k2, v2):
                t[step.lists[b][at // 64], :, at % 64, ::3] = fill
        for b in range(2):
            held = past[b] + rows[b]
            for t in (k2, v2):
                t[step.lists[b][held // 64], :, held % 64:] = fill
        from mynah_slm_b200.ops import tree
        out = torch.full_like(clean, 7.0)
        tree.attn_tree(q.to(DEV), out, step, H, KV, HD, k2.to(DEV), v2.to(DEV), step.pages, masks.to(DEV))
        torch.cuda.synchronize()
        at = 0
        for b, row in ((0, 3), (1, 40)):
            for i in range(rows[b]):
                if seen[b][i, past[b] + row]:
                    assert not torch.isfinite(out[at + i].float()).all()
                else:
                    assert torch.equal(out[at + i], clean[at + i]), (fill, b, i)
            at += rows[b]


@pytest.mark.parametrize("HD", [64, 128, 48])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_a_seen_infinity_in_the_values_reaches_just_its_columns(dtype, HD):
    rows, past, H, KV = [30], [40], 4, 2
    step, q, k, v = _case(17, rows, past, H, KV, HD, dtype)
    masks = _masks([_tree(30, random.Random(8))])
    clean = _check(step, q, k, v, H, KV, HD, masks, dtype).view(30, H, HD)
    at = past[0] + 2
    v[step.lists[0][at // 64], 1, at % 64, 5] = float("inf")
    from mynah_slm_b200.ops import tree
    out = torch.zeros((30, H * HD), dtype=dtype, device=DEV)
    tree.attn_tree(q.to(DEV), out, step, H, KV, HD, k.to(DEV), v.to(DEV), step.pages, masks.to(DEV))
    out = out.view(30, H, HD)
    sees = plain.by_words(step, masks)[0][:, at].to(DEV)
    want = clean.clone()
    want[:, 2:, 5] = torch.where(sees[:, None], torch.full_like(want[:, 2:, 5], float("inf")), want[:, 2:, 5])
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_wide_rows_rows_behind_the_last_and_a_scale(dtype):
    rows, past, H, KV, HD = [12, 30], [100, 7], 4, 2, 64
    rng = random.Random(2)
    for pad, wide, scale in ((0, 0, 0.3), (5, 64, 0.0), (3, 8, 1.0), (0, 3, 0.0)):     # (3 columns more: rows that are not aligned)
        step, q, k, v = _case(19, rows, past, H, KV, HD, dtype, pad, wide)
        _check(step, q, k, v, H, KV, HD, _masks([_tree(n, rng) for n in rows]), dtype, scale, pad=pad)


def test_a_page_that_is_not_there_is_reported_and_read_by_nobody():
    from mynah_slm_b200.ops import tree
    from mynah_slm_b200.ops.kernels import PageTableView
    for dtype in (BF16, F32):
        rows, past, H, KV, HD = [4, 4], [200, 100], 4, 2, 64
        step, q, k, v = _case(23, rows, past, H, KV, HD, dtype)
        ids = step.pages.ids.clone()
        ids[1] = 1 << 20
        bad = PageTableView(step.pages.indptr, ids, step.pages.base, step.pages.n_pages)
        masks = _masks([[-1, 0, 1, 2]] * 2).to(DEV)
        out = torch.zeros((8, H * HD), dtype=dtype, device=DEV)
        tree.attn_tree(q.to(DEV), out, step, H, KV, HD, k.to(DEV), v.to(DEV), bad, masks)
        torch.cuda.synchronize()
        assert step.status.item() & 1
        step.status.zero_()
        good = torch.zeros_like(out)
        tree.attn_tree(q.to(DEV), good, step, H, KV, HD, k.to(DEV), v.to(DEV), step.pages, masks)
        assert step.status.item() == 0 and torch.equal(out[4:], good[4:])


def test_a_captured_call_serves_other_lengths_and_other_streams():
    from mynah_slm_b200.ops import tree
    for dtype, HD in ((BF16, 128), (F32, 64)):
        H, KV = 4, 2
        rng = random.Random(4)
        steps = [_case(s, rows, past, H, KV, HD, dtype) for s, rows, past in
                 ((1, [6, 20], [500, 90]), (2, [20, 6], [40, 700]), (3, [1, 0], [1000, 0]))]
        pool = max(s[0].pages.n_pages for s in steps)
        T, W = 26, 1
        q = torch.zeros((T, H * HD), dtype=dtype, device=DEV)
        k, v = (torch.zeros((pool, KV, 64, HD), dtype=dtype, device=DEV) for _ in range(2))
        masks = torch.zeros((T, W), dtype=torch.int64, device=DEV)
        from types import SimpleNamespace
        i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
        pages = SimpleNamespace(indptr=i32(3), ids=i32(40), base=i32(2), n_pages=pool)
        ctx = SimpleNamespace(B=2, max_q_len=20, cu_q=i32(3), kv_len=i32(2), status=i32(1))
        out = torch.zeros((T, H * HD), dtype=dtype, device=DEV)
        scratch = torch.empty(tree.attn_tree_scratch_floats(T, 2, 20, H, KV, HD, dtype), device=DEV)

        def load(step, q0, k0, v0, m):
            n = step.pages.n_pages
            q.zero_()
            q[:q0.shape[0]] = q0.to(DEV)
            k[:n], v[:n] = k0.to(DEV), v0.to(DEV)
            masks[:m.shape[0]] = m.to(DEV)
            pages.indptr.copy_(step.pages.indptr)
            pages.ids[:step.pages.ids.numel()] = step.pages.ids
            ctx.cu_q.copy_(step.cu_q)
            ctx.kv_len.copy_(step.kv_len)
        trees = [_masks([_tree(n, rng) for n in s[0].q_lens]) for s in steps]
        load(*steps[0], trees[0])
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            tree.attn_tree(q, out, ctx, H, KV, HD, k, v, pages, masks, scratch=scratch)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                tree.attn_tree(q, out, ctx, H, KV, HD, k, v, pages, masks, scratch=scratch)
        for (step, q0, k0, v0), m in zip(steps, trees):
            load(step, q0, k0, v0, m)
            out.fill_(3.0)
            scratch.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            n = q0.shape[0]
            want = _check(step, q0, k0, v0, H, KV, HD, m, dtype)
            rel = (out[:n].double() - want.double()).norm() / want.double().norm()
            assert rel <= (2 * 2.0 ** -8 if dtype == BF16 else 1e-5)       # (chunks may be cut elsewhere: other roundings)
            assert (out[n:] == 3.0).all()


def test_attn_tree_refuses():
    from mynah_slm_b200.ops import tree
    from mynah_slm_b200.ops.lib import KernelError
    H, KV, HD = 4, 2, 64
    step, q, k, v = _case(29, [4], [70], H, KV, HD, BF16)
    q, k, v = q.to(DEV), k.to(DEV), v.to(DEV)
    m = _masks([[-1, 0, 0, 1]]).to(DEV)
    out = torch.zeros_like(q)

    def bad(**kw):
        a = dict(q=q, out=out, ctx=step, H=H, KV=KV, HD=HD, k_cache=k, v_cache=v, pages=step.pages, masks=m, scale=0.0)
        a.update(kw)
        with pytest.raises(KernelError):
            tree.attn_tree(**a)
    bad(q=q.cpu())
    bad(q=q.half(), out=out.half())
    bad(q=q.float())
    bad(out=out[:2])
    bad(q=q[:, ::2])
    bad(out=q)
    bad(H=3)
    bad(KV=0)
    bad(HD=60)
    bad(k_cache=k[:, :1])
    bad(k_cache=k.float())
    bad(v_cache=v[:2])
    bad(v_cache=v.transpose(1, 2).contiguous().transpose(1, 2))
    bad(masks=m.int())
    bad(masks=m[:2])
    bad(masks=m[:, :0])
    bad(scale=-1.0)
    bad(scale=float("nan"))
    bad(scratch=torch.empty(1, device=DEV))
    bad(scratch=torch.empty(100000, device=DEV, dtype=torch.float64))
    tree.attn_tree(q[:0], out[:0], step, H, KV, HD, k, v, step.pages, m[:0])   # nothing to do
    assert (out == 0).all()


# ---------------------------------------------------------------- acceptance

def _commit_case(seed, rows, past, E, KV, HD, VD, dtype, hit=0.85, vocab=50):
    g, rng = _gen(seed), random.Random(seed)
    step = plain.make_step(rows, past, DEV, g)
    k = torch.randn((E, step.pages.n_pages, KV, 64, HD), generator=g).to(dtype)
    v = torch.randn((E, step.pages.n_pages, KV, 64, VD), generator=g).to(dtype)
    tokens, parents, chosen = [], [], []
    for n in rows:
        p = _tree(n, rng)
        t = [rng.randrange(vocab) for _ in range(n)]
        c = [rng.randrange(vocab) for _ in range(n)]
        for i in range(n):
            kids = [j for j in range(n) if p[j] == i]
            if kids and rng.random() < hit:
                c[i] = t[rng.choice(kids)]
        tokens.append(t), parents.append(p), chosen.append(c)
    return step, k, v, tokens, parents, chosen


@pytest.mark.parametrize("rows,past,E,KV,HD,VD,dtype", [
    ([8], [100], 2, 2, 128, 128, BF16), ([1], [0], 1, 1, 64, 64, F32), ([64, 3, 0, 20], [60, 63, 5, 200], 3, 4, 64, 64, BF16),
    ([40, 100], [1, 30], 5, 3, 48, 32, F32), ([300], [17], 2, 2, 8, 16, BF16), ([12] * 40, list(range(40)), 2, 2, 64, 64, BF16),
    ([200], [63], 1, 1, 24, 40, BF16),
])
def test_commit_moves_the_accepted_path(rows, past, E, KV, HD, VD, dtype):
    from mynah_slm_b200.ops import tree
    for seed, hit in ((1, 0.9), (2, 1.0), (3, 0.3)):
        step, k, v, tokens, parents, chosen = _commit_case(seed, rows, past, E, KV, HD, VD, dtype, hit)
        flat = lambda x: torch.tensor([i for l in x for i in l], dtype=torch.int32, device=DEV)  # noqa: E731
        kd, vd = k.to(DEV), v.to(DEV)
        path, count, after = tree.tree_commit(flat(tokens), flat(parents), flat(chosen), step, kd, vd, step.pages)
        torch.cuda.synchronize()
        assert step.status.item() == 0
        at = 0
        k2, v2 = k.clone(), v.clone()
        for b, n in enumerate(rows):
            want, nxt = plain.accepted(tokens[b], parents[b], chosen[b])
            assert path[at:at + n].tolist() == want + [-1] * (n - len(want))
            assert count[b].item() == len(want) and after[b].item() == nxt
            for i, w in enumerate(want):
                s, d = past[b] + w, past[b] + i
                for x, y in ((k, k2), (v, v2)):
                    y[:, step.lists[b][d // 64], :, d % 64] = x[:, step.lists[b][s // 64], :, s % 64]
            at += n
        assert torch.equal(kd.cpu(), k2) and torch.equal(vd.cpu(), v2)


def test_commit_chains_and_odd_parents():
    from mynah_slm_b200.ops import tree
    n = 130
    g = _gen(5)
    step = plain.make_step([n, 6], [50, 10], DEV, g)
    k = torch.randn((2, step.pages.n_pages, 2, 64, 64), generator=g).to(BF16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    # a chain that is accepted whole: nothing moves; a tree whose parents point at rows that are not before them
    tokens = list(range(n)) + [5, 7, 7, 9, 7, 9]
    parents = list(range(-1, n - 1)) + [3, 0, 0, 9, 4, -5]
    chosen = list(range(1, n + 1)) + [7, 9, 9, 9, 9, 9]
    kd, vd = k.to(DEV), k.to(DEV)
    path, count, after = tree.tree_commit(i32(tokens), i32(parents), i32(chosen), step, kd, vd, step.pages)
    assert path[:n].tolist() == list(range(n)) and path[n:].tolist() == [0, 1, -1, -1, -1, -1]
    assert count.tolist() == [n, 2] and after.tolist() == [n, 9]
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), k)
    assert step.status.item() == 0


def test_commit_refuses():
    from types import SimpleNamespace
    from mynah_slm_b200.ops import tree
    from mynah_slm_b200.ops.lib import KernelError
    step, k, v, tokens, parents, chosen = _commit_case(1, [4, 3], [10, 20], 2, 2, 64, 64, BF16)
    k, v = k.to(DEV), v.to(DEV)
    t, p, c = (torch.tensor(x[0] + x[1], dtype=torch.int32, device=DEV) for x in (tokens, parents, chosen))

    def bad(**kw):
        a = dict(tokens=t, parents=p, chosen=c, ctx=step, k_caches=k, v_caches=v, pages=step.pages)
        a.update(kw)
        with pytest.raises(KernelError):
            tree.tree_commit(**a)
    bad(tokens=t.long())
    bad(parents=p[:3])
    bad(chosen=c.cpu())
    bad(k_caches=k[:, :, :1])
    bad(k_caches=k[0])
    bad(v_caches=v.float())
    bad(k_caches=k.cpu())
    long = SimpleNamespace(**{**vars(step), "max_q_len": 5000})
    bad(ctx=long)
    # a longer tree than the step says: refused on the device, the other sequence is served
    short = SimpleNamespace(**{**vars(step), "max_q_len": 3})
    before = k.clone()
    path, count, after = tree.tree_commit(t, p, c, short, k, v, step.pages)
    torch.cuda.synchronize()
    assert count.tolist()[0] == 0 and after.tolist()[0] == -1 and step.status.item() & 1
    want, nxt = plain.accepted(tokens[1], parents[1], chosen[1])
    assert count.tolist()[1] == len(want) and after.tolist()[1] == nxt
    for pg in step.lists[0]:
        assert torch.equal(k[:, pg], before[:, pg])
