"""Attention of a few rows a sequence at lengths and batches where the work is cut in every way (pieces, a line, whole items, several
tiles side by side), caches that pass 32-bit offsets, and calls that run at once; against the definitions in 64 bits."""
import random

import pytest
import torch

from plain import rows as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def _masks(trees):
    from mynah_slm_b200.ops.tree import tree_rows
    words = max(-(-len(t) // 64) for t in trees)
    return torch.cat([torch.from_numpy(tree_rows(t, words)[1].copy()) for t in trees if t])


def _tree(n, rng):
    return [-1 if i == 0 else max(0, i - 1 - int(rng.random() ** 2 * 6)) for i in range(n)]


def _case(seed, rows, past, H, KV, HD, dtype):
    g = torch.Generator().manual_seed(seed)
    step = plain.make_step(rows, past, DEV, g)
    d = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn((sum(rows), H * HD), generator=d, device=DEV).to(dtype)
    k, v = (torch.randn((step.pages.n_pages, KV, 64, HD), generator=d, device=DEV).to(dtype) for _ in range(2))
    return step, q, k, v


def _attention(step, q, k, v, H, scale, sees, p_bits, acc):
    """`plain.attention` for many rows at once: the same formulas and bounds, in 64 bits on the device."""
    KV, HD = k.shape[1], k.shape[3]
    G = H // KV
    out = torch.zeros((q.shape[0], H, HD), dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    sums, room, at = [], [], 0
    for b, (n, p) in enumerate(zip(step.q_lens, step.past)):
        held, pages = p + n, torch.tensor(step.lists[b], device=DEV)
        total, slack = (torch.zeros((KV, held), dtype=torch.float64, device=DEV) for _ in range(2))
        for g in range(KV):
            if n == 0:
                break
            kk, vv = (c[pages, g].reshape(-1, HD)[:held].double() for c in (k, v))
            qq = q[at:at + n, g * G * HD:(g + 1) * G * HD].double().view(n * G, HD)
            seen = sees[b].to(DEV).repeat_interleave(G, 0)
            w = torch.softmax((qq @ kk.T * scale).masked_fill(~seen, float("-inf")), 1)
            A = (qq.abs() @ kk.abs().T * scale).masked_fill(~seen, 0.0).amax(1, keepdim=True)
            N = seen.sum(1, keepdim=True)
            rel = (HD + 2) * acc * A * 2 + 8 * acc * (A + 8) + 2.0 ** -20 + (N + 16) * acc
            out[at:at + n, g * G:(g + 1) * G] = (w @ vv).view(n, G, HD)
            bound[at:at + n, g * G:(g + 1) * G] = ((w @ vv.abs()) * (rel + p_bits + N * acc)).view(n, G, HD)
            total[g], slack[g] = w.sum(0), (w * (rel + (n * G + 4) * acc)).sum(0)
        sums.append(total)
        room.append(slack)
        at += n
    return out, bound, sums, room


def _agrees(step, q, k, v, H, KV, HD, dtype, out, sees, mass=None, got=None):
    tc = dtype == BF16 and HD in (64, 128)
    ref, bound, sums, slack = _attention(step, q, k, v, H, HD ** -0.5, sees, 2.0 ** -8 if tc else 0.0, 2 * plain.F32 if tc else plain.F32)
    last = 2.0 ** -8 if dtype == BF16 else plain.F32
    tol = bound + last * (ref.abs() + bound) + 1e-37
    off = (out.double().view(ref.shape) - ref).abs()
    assert (off <= tol).all(), f"worst {float((off / tol).nan_to_num(1e9).max()):.2f} of the bound"
    if mass is None:
        return
    want, room = mass.double().clone(), torch.zeros(mass.shape, dtype=torch.float64, device=DEV)
    for b, (n, p) in enumerate(zip(step.q_lens, step.past)):
        if n == 0:
            continue
        held, pages = p + n, torch.tensor(step.lists[b], device=DEV)
        r = torch.arange(held, device=DEV)
        at = (pages[r // 64], slice(None), r % 64)
        old = torch.where((r < p)[:, None], mass[at].double(), 0.0)
        want[at] = old + sums[b].T
        room[at] = slack[b].T + plain.F32 * 4 * want[at]
    off = (got.double() - want).abs()
    assert (off <= room).all(), f"sums: worst {float((off / (room + 1e-300)).nan_to_num(1e9).max()):.2f} of the bound"


TREES = [  # rows, past, H, KV, HD: what is cut
    ([8] + [6] * 15, [6000] + [300] * 15, 8, 4, 128),                       # a line under 32 sequences
    ([1 + b % 9 for b in range(45)], [(b * 397) % 2100 for b in range(45)], 8, 2, 64),      # a line of more than 32
    ([200, 90, 0, 256], [3000, 700, 50, 64], 8, 2, 128),                    # tiles by twos, side by side
    ([300, 10], [129, 2000], 16, 2, 64),
    ([600], [1500], 8, 1, 128),                                             # five tiles, and ten words of masks
    ([8], [30000], 4, 1, 128),                                              # one item, a piece a CTA
    ([2, 3], [20000, 64], 1, 1, 64),
    ([5, 2], [300, 70], 100, 1, 64),                                        # a token a tile
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", TREES, ids=lambda c: f"{len(c[0])}seq-{c[0][0]}x{c[1][0]}-{c[2]}:{c[3]}x{c[4]}")
def test_tree_attention_however_it_is_cut(case, dtype):
    from mynah_slm_b200.ops import tree
    rows, past, H, KV, HD = case
    rng = random.Random(len(rows))
    step, q, k, v = _case(2, rows, past, H, KV, HD, dtype)
    masks = _masks([_tree(n, rng) for n in rows])
    out = torch.zeros_like(q)
    tree.attn_tree(q, out, step, H, KV, HD, k, v, step.pages, masks.to(DEV))
    assert step.status.item() == 0
    sees, at = [], 0
    for n, p in zip(rows, past):
        j = torch.arange(n)
        own = ((masks[at:at + n][:, j // 64] >> (j % 64)) & 1).bool() if n else torch.zeros((0, 0), dtype=torch.bool)
        sees.append(torch.cat([torch.ones((n, p), dtype=torch.bool), own], 1))
        at += n
    _agrees(step, q, k, v, H, KV, HD, dtype, out, sees)


@pytest.mark.parametrize("dtype,HD", [(BF16, 64), (BF16, 128), (BF16, 48), (F32, 64)], ids=["tc64", "tc128", "bf16-48", "f32"])
def test_missing_pages_where_a_cta_has_several_segments(dtype, HD):
    """Pages that are not there, in sequences of a long ragged batch (a CTA's share of it reaches over several of them): reported, read by
    nobody, and every other sequence has the bits that it has without them."""
    from mynah_slm_b200.ops import tree
    from mynah_slm_b200.ops.kernels import PageTableView
    rows, past, H, KV = [1 + b % 9 for b in range(45)], [(b * 397) % 2100 for b in range(45)], 8, 2
    rng = random.Random(45)
    step, q, k, v = _case(12, rows, past, H, KV, HD, dtype)
    masks = _masks([_tree(n, rng) for n in rows]).to(DEV)
    want = torch.zeros_like(q)
    tree.attn_tree(q, want, step, H, KV, HD, k, v, step.pages, masks)
    assert step.status.item() == 0
    indptr = step.pages.indptr.tolist()
    lacking = [b for b in range(45) if b % 4 == 1]
    ids = step.pages.ids.clone()
    for b in lacking:
        ids[indptr[b] + rng.randrange(indptr[b + 1] - indptr[b])] = rng.choice([-1, -3, step.pages.n_pages, 1 << 20])
    bad = PageTableView(step.pages.indptr, ids, step.pages.base, step.pages.n_pages)
    for _ in range(5):
        out = torch.full_like(q, 7.0)
        tree.attn_tree(q, out, step, H, KV, HD, k, v, bad, masks)
        assert step.status.item() & 1 and step.status.item() & 16 == 0
        step.status.zero_()
        at = 0
        for b, n in enumerate(rows):
            if b not in lacking:
                assert torch.equal(out[at:at + n], want[at:at + n]), b
            at += n


STEPS = [
    ([700, 1500, 40], [0, 100, 900], 16, 8, 128),                           # whole items
    ([300, 5, 1], [4000, 50, 9], 4, 2, 128),                                # several tiles of different lengths on a line
    ([20] * 40, [(b * 211) % 900 for b in range(40)], 8, 2, 64),            # more than 32 sequences, sums by keys
    ([1] * 50, [(b * 631) % 4000 for b in range(50)], 8, 2, 128),           # sums from kept scores
    ([1], [40000], 8, 1, 64),
    ([90, 33], [5000, 2], 10, 2, 128),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", STEPS, ids=lambda c: f"{len(c[0])}seq-{c[0][0]}x{c[1][0]}-{c[2]}:{c[3]}x{c[4]}")
def test_sums_however_they_are_cut(case, dtype):
    from mynah_slm_b200.ops import evict
    rows, past, H, KV, HD = case
    step, q, k, v = _case(3, rows, past, H, KV, HD, dtype)
    mass = torch.rand((step.pages.n_pages, KV, 64), device=DEV) * 3
    got, out = mass.clone(), torch.zeros_like(q)
    evict.attn_mass(q, out, got, step, H, KV, HD, k, v, step.pages)
    assert step.status.item() == 0
    _agrees(step, q, k, v, H, KV, HD, dtype, out, plain.causal(step), mass, got)


def test_scales_that_fp32_does_not_hold_are_refused():
    """One that rounds to 0 there would have been taken for "not given"."""
    from mynah_slm_b200.ops import evict, tree
    from mynah_slm_b200.ops.lib import KernelError
    H, KV, HD = 4, 2, 64
    step, q, k, v = _case(5, [2], [70], H, KV, HD, F32)
    mass, out, masks = torch.zeros((step.pages.n_pages, KV, 64), device=DEV), torch.zeros_like(q), _masks([[-1, 0]]).to(DEV)
    for scale in (1e-46, 1e-40, -0.125, 1e38, 1e300, float("inf"), float("nan")):
        with pytest.raises(KernelError):
            tree.attn_tree(q, out, step, H, KV, HD, k, v, step.pages, masks, scale)
        with pytest.raises(KernelError):
            evict.attn_mass(q, out, mass, step, H, KV, HD, k, v, step.pages, scale)
    assert (out == 0).all() and (mass == 0).all()
    small = torch.zeros_like(q)                            # a scale that leaves no difference between the rows: their mean
    tree.attn_tree(q, small, step, H, KV, HD, k, v, step.pages, masks, 2.0 ** -100)
    rows = torch.cat([v[p] for p in step.lists[0]], 1)
    want = torch.stack([rows[:, :n].double().mean(1).repeat_interleave(H // KV, 0) for n in (71, 72)]).view(2, H * HD)
    assert ((small.double() - want).abs() <= 200 * plain.F32 * rows.abs().max()).all() and step.status.item() == 0


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_an_output_over_q_is_refused_and_one_beside_it_served(dtype):
    from mynah_slm_b200.ops import evict, tree
    from mynah_slm_b200.ops.lib import KernelError
    rows, past, H, KV, HD = [9, 4], [100, 30], 4, 2, 64
    step, q, k, v = _case(8, rows, past, H, KV, HD, dtype)
    W, T = H * HD, sum(rows)
    masks, mass = _masks([[-1] + list(range(n - 1)) for n in rows]).to(DEV), torch.zeros((step.pages.n_pages, KV, 64), device=DEV)
    wide = torch.zeros((T + 1, 3 * W), dtype=dtype, device=DEV)
    wide[:T, :W] = q
    for out in (wide[1:, :W], wide[:T, 8:W + 8], wide[:T, W - 8:2 * W - 8], wide.view(-1)[W // 2:W // 2 + T * W].view(T, W)):
        with pytest.raises(KernelError):
            tree.attn_tree(wide[:T, :W], out, step, H, KV, HD, k, v, step.pages, masks)
        with pytest.raises(KernelError):
            evict.attn_mass(wide[:T, :W], out, mass, step, H, KV, HD, k, v, step.pages)
    assert torch.equal(wide[:T, :W], q) and (wide[:, W:] == 0).all() and (mass == 0).all()
    want = torch.zeros_like(q)
    tree.attn_tree(q, want, step, H, KV, HD, k, v, step.pages, masks)
    for out in (wide[:T, W:2 * W], wide[1:, W:2 * W], wide[:T, 2 * W:]):
        tree.attn_tree(wide[:T, :W], out, step, H, KV, HD, k, v, step.pages, masks)
        assert torch.equal(out, want) and torch.equal(wide[:T, :W], q)
    assert step.status.item() == 0


COMPANY = [  # a sequence's rows and past, then the others' in every company
    (1, 1535, [([1], [40]), ([1] * 5, [6000, 3, 64, 900, 2047]), ([1] * 63, [(b * 631) % 4000 for b in range(63)]),
               ([1] * 300, [(b * 37) % 300 for b in range(300)])]),
    (1, 63, [([1] * 9, [9000] * 9), ([300, 9], [200, 64]), ([17, 1, 0, 2], [5, 70, 90, 400])]),           # (and tiles of another size)
    (5, 700, [([1, 3], [64, 2000]), ([200], [0])]),
    (40, 700, [([33], [10]), ([300, 9], [2000, 64]), ([12] * 40, [(b * 211) % 900 for b in range(40)])]),
    (150, 333, [([150], [333]), ([64, 170], [3000, 5]), ([60] * 10, [500] * 10)]),
]


@pytest.mark.parametrize("dtype,H,KV,HD", [(BF16, 6, 2, 48), (BF16, 16, 8, 80), (F32, 8, 2, 64), (F32, 4, 4, 128), (F32, 32, 8, 128)],
                         ids=["bf16-48", "bf16-80", "f32-64", "f32-128", "f32-32on8"])
@pytest.mark.parametrize("case", COMPANY, ids=lambda c: f"{c[0]}x{c[1]}")
def test_a_sequence_has_the_same_bits_in_any_company(case, dtype, H, KV, HD):
    """In 32 bits (and for heads that the tensor cores do not take) outputs and sums do not depend on what else the step brings, and
    with them the path that a tree takes and the rows that an eviction keeps."""
    from mynah_slm_b200.ops import evict, tree
    n, p, companies = case
    d = torch.Generator(device=DEV).manual_seed(77)
    pages = -(-(n + p) // 64)
    own = [torch.randn(shape, generator=d, device=DEV).to(dtype) for shape in ((n, H * HD), (pages, KV, 64, HD), (pages, KV, 64, HD))]
    sums = torch.rand((pages, KV, 64), generator=d, device=DEV) * 3
    mine_tree = _tree(n, random.Random(n))

    def run(rows, past, at):
        rng = random.Random(at)
        step, q, k, v = _case(len(rows), rows, past, H, KV, HD, dtype)
        masks = _masks([mine_tree if b == at else _tree(r, rng) for b, r in enumerate(rows)])
        mine, first = torch.tensor(step.lists[at], device=DEV), sum(rows[:at])
        mass = torch.rand((step.pages.n_pages, KV, 64), device=DEV) * 3
        q[first:first + n], k[mine], v[mine], mass[mine] = own[0], own[1], own[2], sums
        out, hung = torch.zeros_like(q), torch.zeros_like(q)
        evict.attn_mass(q, out, mass, step, H, KV, HD, k, v, step.pages)
        tree.attn_tree(q, hung, step, H, KV, HD, k, v, step.pages, masks.to(DEV))
        assert step.status.item() == 0
        return out[first:first + n].clone(), mass[mine].clone(), hung[first:first + n].clone()
    alone = run([n], [p], 0)
    for rows, past in companies:
        for at in sorted({0, len(rows) // 2, len(rows)}):
            got = run(rows[:at] + [n] + rows[at:], past[:at] + [p] + past[at:], at)
            for a, b, what in zip(got, alone, ("outputs", "sums", "tree")):
                assert torch.equal(a, b), (len(rows), at, what)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,past,most", [([1, 1, 3], [200, 63, 500], 1), ([20, 3, 150], [100, 700, 90], 20), ([130, 3, 131], [0, 50, 300], 130)])
def test_a_longer_sequence_than_the_step_says_is_refused(rows, past, most, dtype):
    """The sums are made for max_q_len rows of a sequence: one with more is reported and left alone, the others are served."""
    from types import SimpleNamespace
    from mynah_slm_b200.ops import evict
    H, KV, HD = 4, 2, 64
    step, q, k, v = _case(9, rows, past, H, KV, HD, dtype)
    step.max_q_len = most
    mass = torch.rand((step.pages.n_pages, KV, 64), device=DEV) * 3
    got, out = mass.clone(), torch.full_like(q, 7.0)
    evict.attn_mass(q, out, got, step, H, KV, HD, k, v, step.pages)
    assert step.status.item() & 1
    n = sum(rows[:2])
    assert (out[n:] == 7.0).all()
    served = SimpleNamespace(q_lens=rows[:2], past=past[:2], lists=step.lists[:2])
    _agrees(served, q[:n], k, v, H, KV, HD, dtype, out[:n], plain.causal(served), mass, got)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,past", [([1, 1, 1], [300, 64, 5]), ([40, 7], [30, 200])])
def test_outputs_that_are_not_aligned(rows, past, dtype):
    """Columns of a wider buffer that begin at an odd one, rows of an odd pitch; q is aligned."""
    from mynah_slm_b200.ops import evict, tree
    H, KV, HD = 4, 2, 64
    step, q, k, v = _case(6, rows, past, H, KV, HD, dtype)
    mass = torch.rand((step.pages.n_pages, KV, 64), device=DEV) * 3
    wide = torch.full((sum(rows), H * HD + 3), 7.0, dtype=dtype, device=DEV)
    out, got = wide[:, 1:1 + H * HD], mass.clone()
    evict.attn_mass(q, out, got, step, H, KV, HD, k, v, step.pages)
    assert step.status.item() == 0 and (wide[:, 0] == 7.0).all() and (wide[:, 1 + H * HD:] == 7.0).all()
    tight = out.contiguous()
    _agrees(step, q, k, v, H, KV, HD, dtype, tight, plain.causal(step), mass, got)
    chain = [[-1] + list(range(n - 1)) for n in rows]
    tree.attn_tree(q, out, step, H, KV, HD, k, v, step.pages, _masks(chain).to(DEV))
    _agrees(step, q, k, v, H, KV, HD, dtype, out.contiguous(), plain.causal(step))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_a_step_of_nothing_but_padding(dtype):
    """Sequences without rows in the step, and rows of q behind the last one: nothing is written."""
    from mynah_slm_b200.ops import evict, tree
    H, KV, HD = 4, 2, 64
    step, _, k, v = _case(4, [0, 0], [100, 0], H, KV, HD, dtype)
    q, out = torch.randn((6, H * HD), device=DEV).to(dtype), torch.full((6, H * HD), 7.0, dtype=dtype, device=DEV)
    mass = torch.rand((step.pages.n_pages, KV, 64), device=DEV)
    before = mass.clone()
    tree.attn_tree(q, out, step, H, KV, HD, k, v, step.pages, torch.zeros((6, 1), dtype=torch.int64, device=DEV))
    evict.attn_mass(q, out, mass, step, H, KV, HD, k, v, step.pages)
    assert step.status.item() == 0 and (out == 7.0).all() and torch.equal(mass, before)
    ids = torch.zeros(6, dtype=torch.int32, device=DEV)
    path, count, after = tree.tree_commit(ids, ids, ids, step, k[None], v[None], step.pages)
    assert step.status.item() == 0 and count.tolist() == [0, 0] and after.tolist() == [-1, -1]


def test_caches_that_pass_32_bit_offsets():
    """2,150 pages of 128 kv heads: 2.25 * 10^9 values. The sequences lie in the last pages and in the first ones."""
    from mynah_slm_b200.ops import evict, tree
    KV, HD, n_pages, rows, past = 128, 128, 2150, [5, 3], [300, 200]
    g = torch.Generator().manual_seed(1)
    lists = [[n_pages - 1 - i for i in range(5)], [3, 0, n_pages - 9, 7]]
    step = plain.make_step(rows, past, DEV, g, lists=lists)
    step.pages.n_pages = n_pages
    used = sorted(p for l in lists for p in l)
    k, v = (torch.empty((n_pages, KV, 64, HD), dtype=BF16, device=DEV) for _ in range(2))
    d = torch.Generator(device=DEV).manual_seed(1)
    for p in used:
        for c in (k, v):
            c[p] = torch.randn((KV, 64, HD), generator=d, device=DEV).to(BF16)
    q = torch.randn((8, KV * HD), generator=d, device=DEV).to(BF16)
    trees = [[-1, 0, 0, 1, 3], [-1, 0, 1]]
    masks = _masks(trees)
    small = torch.tensor(used, device=DEV)
    where = {p: i for i, p in enumerate(used)}
    near = plain.make_step(rows, past, DEV, g, lists=[[where[p] for p in l] for l in lists])
    near.pages.n_pages = len(used)
    kn, vn = k[small].contiguous(), v[small].contiguous()
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    tree.attn_tree(q, out, step, KV, KV, HD, k, v, step.pages, masks.to(DEV))
    tree.attn_tree(q, want, near, KV, KV, HD, kn, vn, near.pages, masks.to(DEV))
    assert step.status.item() == 0 and torch.equal(out, want)
    mass = torch.rand((n_pages, KV, 64), device=DEV)
    mn = mass[small].contiguous()
    evict.attn_mass(q, out, mass, step, KV, KV, HD, k, v, step.pages)
    evict.attn_mass(q, want, mn, near, KV, KV, HD, kn, vn, near.pages)
    assert step.status.item() == 0 and torch.equal(out, want) and torch.equal(mass[small], mn)
    tokens = torch.tensor([9, 4, 5, 6, 7, 1, 2, 3], dtype=torch.int32, device=DEV)
    parents = torch.tensor(trees[0] + trees[1], dtype=torch.int32, device=DEV)
    chosen = torch.tensor([5, 0, 8, 0, 0, 2, 3, 4], dtype=torch.int32, device=DEV)
    far = tree.tree_commit(tokens, parents, chosen, step, k[None], v[None], step.pages)
    ref = tree.tree_commit(tokens, parents, chosen, near, kn[None], vn[None], near.pages)
    assert all(torch.equal(a, b) for a, b in zip(far, ref)) and far[1].tolist() == [2, 3]
    assert torch.equal(k[small], kn) and torch.equal(v[small], vn)
    kept, after = evict.cache_evict(k[None], v[None], mass[None], step, step.pages, 150, 40, 3)
    kept_n, after_n = evict.cache_evict(kn[None], vn[None], mn[None], near, near.pages, 150, 40, 3)
    assert step.status.item() == 0 and torch.equal(kept, kept_n) and torch.equal(after, after_n)
    assert torch.equal(k[small], kn) and torch.equal(v[small], vn) and torch.equal(mass[small], mn)


def test_calls_at_once_on_two_streams_and_two_graphs():
    """Every call has a workspace of its own: calls that run at once, and graphs captured one after the other and replayed at once,
    give the bits that each gives alone."""
    from mynah_slm_b200.ops import evict, tree
    H, KV, HD = 8, 4, 128
    rng = random.Random(5)
    jobs = []
    for s, (rows, past) in enumerate((([24] * 4, [1500, 900, 30, 2000]), ([8] * 8, [700] * 8))):
        step, q, k, v = _case(30 + s, rows, past, H, KV, HD, BF16)
        masks = _masks([_tree(n, rng) for n in rows]).to(DEV)
        mass = torch.rand((step.pages.n_pages, KV, 64), device=DEV)

        def run(step=step, q=q, k=k, v=v, masks=masks, mass=mass):
            a, b, m = torch.zeros_like(q), torch.zeros_like(q), mass.clone()
            tree.attn_tree(q, a, step, H, KV, HD, k, v, step.pages, masks)
            evict.attn_mass(q, b, m, step, H, KV, HD, k, v, step.pages)
            return a, b, m
        jobs.append((run, [t.clone() for t in run()], step))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(10):
        got = []
        for (run, _, _), st in zip(jobs, streams):
            with torch.cuda.stream(st):
                got.append(run())
        torch.cuda.synchronize()
        for outs, (_, want, step) in zip(got, jobs):
            assert step.status.item() == 0 and all(torch.equal(x, y) for x, y in zip(outs, want))
    graphs = []
    for (run, _, _), st in zip(jobs, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs = run()
        graphs.append((graph, outs))
    for _ in range(10):
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for (_, outs), (_, want, step) in zip(graphs, jobs):
            assert step.status.item() == 0 and all(torch.equal(x, y) for x, y in zip(outs, want))


def test_a_captured_eviction_and_acceptance_serve_other_lengths():
    """One graph of an acceptance and an eviction; its replays go by the lengths, trees and choices of the moment."""
    from mynah_slm_b200.ops import evict, tree
    E, KV, HD, rows = 3, 2, 64, [6, 4]
    g = torch.Generator().manual_seed(3)
    step = plain.make_step(rows, [700, 400], DEV, g)
    d = torch.Generator(device=DEV).manual_seed(3)
    shape = (E, step.pages.n_pages, KV, 64)
    k, v = (torch.randn((*shape, HD), generator=d, device=DEV).to(BF16) for _ in range(2))
    mass = torch.rand(shape, generator=d, device=DEV)
    tokens, parents, chosen = (torch.zeros(10, dtype=torch.int32, device=DEV) for _ in range(3))

    def run(k, v, mass):
        moved = tree.tree_commit(tokens, parents, chosen, step, k, v, step.pages)
        return [*moved, *evict.cache_evict(k, v, mass, step, step.pages, 200, 50, 4)]
    side = torch.cuda.Stream()
    kg, vg, mg = k.clone(), v.clone(), mass.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = run(kg, vg, mg)
    rng = random.Random(8)
    for held in ([706, 404], [650, 150], [200, 201], [6, 4]):
        step.kv_len.copy_(torch.tensor(held, dtype=torch.int32))
        trees = [_tree(n, rng) for n in rows]
        parents.copy_(torch.tensor(trees[0] + trees[1], dtype=torch.int32))
        tokens.copy_(torch.tensor([rng.randrange(3) for _ in range(10)], dtype=torch.int32))
        chosen.copy_(torch.tensor([rng.randrange(3) for _ in range(10)], dtype=torch.int32))
        for a, b in ((kg, k), (vg, v), (mg, mass)):
            a.copy_(b)
        ke, ve, me = k.clone(), v.clone(), mass.clone()
        want = run(ke, ve, me)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert step.status.item() == 0
        assert all(torch.equal(a, b) for a, b in zip([*outs, kg, vg, mg], [*want, ke, ve, me]))
        assert outs[4].tolist() == [min(h, 200) for h in held]
        for b, n in enumerate(rows):
            at = sum(rows[:b])
            path, nxt = plain.accepted(tokens[at:at + n].tolist(), trees[b], chosen[at:at + n].tolist())
            assert outs[1].tolist()[b] == len(path) and outs[2].tolist()[b] == nxt and outs[0].tolist()[at:at + len(path)] == path
