"""Attention that adds up the cached rows' weights, and the eviction by them, against the definitions in 64 bits."""
import random

import pytest
import torch

from plain import rows as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _case(seed, rows, past, H, KV, HD, dtype, pad=0, wide=0):
    g = _gen(seed)
    step = plain.make_step(rows, past, DEV, g)
    q = torch.randn((sum(rows) + pad, H * HD + wide), generator=g).to(dtype)
    k = torch.randn((step.pages.n_pages, KV, 64, HD), generator=g).to(dtype)
    v = torch.randn((step.pages.n_pages, KV, 64, HD), generator=g).to(dtype)
    mass = torch.rand((step.pages.n_pages, KV, 64), generator=g) * 3
    return step, q, k, v, mass


def _tensor_cores(dtype, H, KV, HD):
    return dtype == BF16 and HD in (64, 128) and H // KV <= 128


def _check(step, q, k, v, mass, H, KV, HD, dtype, scale=0.0):
    from mynah_slm_b200.ops import evict
    n = sum(step.q_lens)
    out = torch.full((q.shape[0], H * HD), 7.0, dtype=dtype, device=DEV)
    md = mass.to(DEV)
    evict.attn_mass(q.to(DEV), out, md, step, H, KV, HD, k.to(DEV), v.to(DEV), step.pages, scale)
    torch.cuda.synchronize()
    assert step.status.item() == 0
    tc = _tensor_cores(dtype, H, KV, HD)
    ref, bound, sums, slack = plain.attention(step, q[:, :H * HD], k, v, H, scale or HD ** -0.5, plain.causal(step),
                                              2.0 ** -8 if tc else 0.0, 2 * plain.F32 if tc else plain.F32)
    ref, bound = ref[:n], bound[:n]
    o = out[:n].double().cpu().view(n, H, HD)
    last = 2.0 ** -8 if dtype == BF16 else plain.F32
    tol = bound + last * (ref.abs() + bound) + 1e-37
    bad = ~((o - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values, worst {float(((o - ref).abs() / tol).nan_to_num(1e9).max()):.2f} of the bound"
    assert (out[n:] == 7.0).all(), "rows behind the last sequence"
    want, room = mass.double().clone(), torch.zeros(mass.shape, dtype=torch.float64)
    for b, (nq, p) in enumerate(zip(step.q_lens, step.past)):
        if nq == 0:
            continue                                       # a sequence that is not in the step keeps its sums
        for r in range(p + nq):
            at = (step.lists[b][r // 64], slice(None), r % 64)
            old = mass[at].double() if r < p else 0.0
            want[at] = old + sums[b][:, r]
            room[at] = slack[b][:, r] + plain.F32 * 4 * want[at]
    bad = ~((md.double().cpu() - want).abs() <= room)
    assert not bad.any(), f"sums: {int(bad.sum())} of {bad.numel()}, worst off {float((md.double().cpu() - want).abs().max()):.3e}"
    return out, md


CASES = [  # rows, past, H, KV, HD
    ([1], [0], 2, 1, 64), ([1], [1], 4, 2, 128), ([1], [63], 16, 8, 128), ([1] * 6, [64, 65, 700, 0, 127, 200], 8, 2, 128),
    ([1] * 40, list(range(10, 410, 10)), 4, 2, 64), ([1], [2000], 2, 2, 128), ([5], [60], 4, 2, 64), ([64], [0], 4, 2, 64),
    ([65], [63], 6, 2, 128), ([130, 1, 0, 200], [1, 300, 50, 0], 4, 2, 64), ([257], [129], 2, 1, 128), ([300], [0], 3, 1, 64),
    ([90, 20], [70, 5], 12, 4, 48), ([7], [100], 5, 5, 8), ([40], [33], 6, 3, 80), ([20], [100], 4, 1, 256), ([3], [90], 40, 1, 64),
    ([2], [70], 200, 1, 64), ([4] * 9, [500] * 9, 4, 4, 128), ([33], [95], 10, 2, 64), ([1], [150], 6, 2, 64),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}seq-{c[0][0]}x{c[1][0]}-{c[2]}:{c[3]}x{c[4]}")
def test_mass_is_the_formula(case, dtype):
    rows, past, H, KV, HD = case
    _check(*_case(3, rows, past, H, KV, HD, dtype), H, KV, HD, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_wide_rows_rows_behind_the_last_and_a_scale(dtype):
    H, KV, HD = 4, 2, 64
    for rows, past in (([12, 30], [100, 7]), ([1, 1], [100, 7])):
        for pad, wide, scale in ((0, 0, 0.3), (5, 64, 0.0), (3, 8, 1.0), (0, 3, 0.0)):
            _check(*_case(19, rows, past, H, KV, HD, dtype, pad, wide), H, KV, HD, dtype, scale)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,past", [([1], [70]), ([40], [50])])
def test_rows_behind_the_last_and_later_rows_have_no_influence(rows, past, dtype):
    from mynah_slm_b200.ops import evict
    H, KV, HD = 4, 2, 64
    step, q, k, v, mass = _case(5, rows, past, H, KV, HD, dtype)
    out, sums = _check(step, q, k, v, mass, H, KV, HD, dtype)
    held = rows[0] + past[0]
    for fill in (float("nan"), float("inf")):
        k2, v2, m2 = k.clone(), v.clone(), mass.clone()
        for t in (k2, v2, m2):
            t[step.lists[0][held // 64], :, held % 64:] = fill
        for r in range(past[0], held):                     # the sums of the step's own rows are not read
            m2[step.lists[0][r // 64], :, r % 64] = fill
        if rows[0] > 1:                                    # the last row is seen by itself alone
            for t in (k2, v2):
                t[step.lists[0][(held - 1) // 64], :, (held - 1) % 64] = fill
        o, md = torch.zeros_like(out), m2.to(DEV)
        evict.attn_mass(q.to(DEV), o, md, step, H, KV, HD, k2.to(DEV), v2.to(DEV), step.pages)
        n = rows[0] - (1 if rows[0] > 1 else 0)
        assert torch.equal(o[:n], out[:n])
        for r in range(held):
            got, want = md[step.lists[0][r // 64], :, r % 64], sums[step.lists[0][r // 64], :, r % 64]
            if rows[0] == 1:
                assert torch.equal(got, want)
        for r in range(held, -(-held // 64) * 64):         # rows behind the last keep what they hold
            a, b = md[step.lists[0][r // 64], :, r % 64].cpu(), m2[step.lists[0][r // 64], :, r % 64]
            assert torch.equal(torch.nan_to_num(a, 9.0), torch.nan_to_num(b, 9.0))


def test_the_sums_do_not_depend_on_timing_and_steps_add_up():
    """The same call gives the same bits; a prompt in pieces and then tokens one by one gives the sums of one long step."""
    from mynah_slm_b200.ops import evict
    H, KV, HD = 4, 2, 64
    for dtype, tol in ((F32, 1e-5), (BF16, 1e-5)):
        step, q, k, v, mass = _case(7, [200], [0], H, KV, HD, dtype)
        first = _check(step, q, k, v, mass, H, KV, HD, dtype)
        again = _check(step, q, k, v, mass, H, KV, HD, dtype)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        md = mass.to(DEV)
        at = 0
        for n in (70, 1, 1, 100, 1, 27):
            part = plain.make_step([n], [at], DEV, _gen(1), lists=[step.lists[0][: -(-(at + n) // 64)]])
            part.pages.n_pages = step.pages.n_pages
            out = torch.zeros((n, H * HD), dtype=dtype, device=DEV)
            evict.attn_mass(q[at:at + n].to(DEV), out, md, part, H, KV, HD, k.to(DEV), v.to(DEV), part.pages)
            assert part.status.item() == 0
            at += n
        rows = [md[step.lists[0][r // 64], :, r % 64] for r in range(200)]
        want = [first[1][step.lists[0][r // 64], :, r % 64] for r in range(200)]
        a, b = torch.stack(rows).double(), torch.stack(want).double()
        assert ((a - b).abs() <= tol * b + 1e-6).all()
        assert abs(a.sum().item() - 200 * H) < 1e-2


def test_a_page_that_is_not_there_is_reported():
    from mynah_slm_b200.ops import evict
    from mynah_slm_b200.ops.kernels import PageTableView
    H, KV, HD = 4, 2, 64
    for dtype in (BF16, F32):
        for rows in ([1, 1], [30, 40]):
            step, q, k, v, mass = _case(9, rows, [200, 150], H, KV, HD, dtype)
            ids = step.pages.ids.clone()
            ids[2] = -7
            bad = PageTableView(step.pages.indptr, ids, step.pages.base, step.pages.n_pages)
            out = torch.zeros((sum(rows), H * HD), dtype=dtype, device=DEV)
            evict.attn_mass(q.to(DEV), out, mass.to(DEV), step, H, KV, HD, k.to(DEV), v.to(DEV), bad)
            torch.cuda.synchronize()
            assert step.status.item() & 1


def test_attn_mass_refuses():
    from mynah_slm_b200.ops import evict
    from mynah_slm_b200.ops.lib import KernelError
    H, KV, HD = 4, 2, 64
    step, q, k, v, mass = _case(29, [4], [70], H, KV, HD, BF16)
    q, k, v, mass = q.to(DEV), k.to(DEV), v.to(DEV), mass.to(DEV)
    out = torch.zeros_like(q)

    def bad(**kw):
        a = dict(q=q, out=out, mass=mass, ctx=step, H=H, KV=KV, HD=HD, k_cache=k, v_cache=v, pages=step.pages, scale=0.0)
        a.update(kw)
        with pytest.raises(KernelError):
            evict.attn_mass(**a)
    bad(mass=mass.double())
    bad(mass=mass[:1])
    bad(mass=mass.cpu())
    bad(mass=mass[:, :1])
    bad(out=out.float())
    bad(HD=12)
    bad(scale=float("inf"))
    bad(scratch=torch.empty(8, device=DEV))


# ------------------------------------------------------------------ eviction

def _evict_case(seed, held, E, KV, HD, VD, dtype, out_rows=0, kind="spread"):
    from mynah_slm_b200.ops.kernels import PageTableView
    g = _gen(seed)
    B = len(held)
    step = plain.make_step([0] * B, held, DEV, g, spare=2 + B * -(-out_rows // 64))
    n = step.pages.n_pages
    k = torch.randn((E, n, KV, 64, HD), generator=g).to(dtype)
    v = torch.randn((E, n, KV, 64, VD), generator=g).to(dtype)
    m = torch.rand((E, n, KV, 64), generator=g) ** 6 * 40
    if kind == "ties":
        m = (m * 0.1).round()
    elif kind == "equal":
        m = torch.full_like(m, 0.25)
    elif kind == "odd":                                    # zeros of both signs, infinities, NaN, negative and tiny sums
        odd = torch.tensor([0.0, -0.0, float("inf"), float("nan"), -1.0, 1e-40, -float("inf"), 2.0])
        m = odd[torch.randint(0, 8, m.shape, generator=g)]
    out = None
    if out_rows:
        used = {p for l in step.lists for p in l}
        free = [p for p in range(n) if p not in used]
        per = -(-out_rows // 64)
        lists = [free[b * per:(b + 1) * per] for b in range(B)]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        out = (PageTableView(i32([per * b for b in range(B + 1)]), i32([p for l in lists for p in l]), i32([0] * B), n), lists)
    return step, k, v, m, out


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("apart", [False, True], ids=["in-place", "apart"])
@pytest.mark.parametrize("held,keep,recent,first,E,KV,HD,VD,dtype", [
    ([700], 512, 64, 4, 1, 2, 128, 128, BF16), ([65], 64, 0, 0, 2, 1, 64, 64, F32), ([300, 20, 0, 130, 64], 64, 10, 3, 3, 2, 64, 64, BF16),
    ([1000, 999], 1, 0, 0, 1, 3, 48, 32, F32), ([500], 100, 60, 40, 2, 2, 8, 16, BF16), ([1500], 1100, 300, 16, 1, 1, 256, 128, F32),
    ([129, 193], 128, 128, 0, 2, 2, 24, 40, BF16), ([2200], 513, 0, 1, 1, 2, 64, 64, BF16), ([90], 89, 5, 5, 1, 4, 128, 64, F32),
])
def test_evict_keeps_the_rows_with_the_greatest_sums(held, keep, recent, first, E, KV, HD, VD, dtype, apart, kind):
    from mynah_slm_b200.ops import evict
    step, k, v, m, out = _evict_case(3, held, E, KV, HD, VD, dtype, keep if apart else 0, kind)
    kd, vd, md = k.to(DEV), v.to(DEV), m.to(DEV)
    kept, n = evict.cache_evict(kd, vd, md, step, step.pages, keep, recent, first, out_pages=out[0] if apart else None)
    torch.cuda.synchronize()
    assert step.status.item() == 0
    assert n.tolist() == [min(h, keep) for h in held]
    k2, v2, m2 = k.clone(), v.clone(), m.clone()
    for b, h in enumerate(held):
        src_pages = torch.tensor(step.lists[b] or [0])
        dst_pages = torch.tensor(out[1][b]) if apart else src_pages
        for e in range(E):
            for g in range(KV):
                sums = m[e, src_pages, g].reshape(-1)[:h].tolist()
                want = plain.kept_rows(sums, h, keep, recent, first)
                assert kept[e, b, g].tolist() == want + [-1] * (keep - len(want)), (b, e, g)
                s, d = torch.tensor(want, dtype=torch.long), torch.arange(len(want))
                for x, y in ((k, k2), (v, v2), (m, m2)):
                    y[e, dst_pages[d // 64], g, d % 64] = x[e, src_pages[s // 64], g, s % 64]
    assert torch.equal(kd.cpu(), k2) and torch.equal(vd.cpu(), v2)
    assert torch.equal(torch.nan_to_num(md.cpu(), 77.0), torch.nan_to_num(m2, 77.0))


def test_evict_of_a_long_sequence():
    """More rows than a CTA keeps the words of."""
    from mynah_slm_b200.ops import evict
    step, k, v, m, _ = _evict_case(5, [30000], 1, 1, 8, 8, BF16)
    kd, vd, md = k.to(DEV), v.to(DEV), m.to(DEV)
    kept, n = evict.cache_evict(kd, vd, md, step, step.pages, 9000, 100, 4)
    pages = torch.tensor(step.lists[0])
    want = plain.kept_rows(m[0, pages, 0].reshape(-1)[:30000].tolist(), 30000, 9000, 100, 4)
    assert kept[0, 0, 0].tolist() == want and n.item() == 9000
    s, d = torch.tensor(want), torch.arange(9000)
    assert torch.equal(kd.cpu()[0, pages[d // 64], 0, d % 64], k[0, pages[s // 64], 0, s % 64])
    assert torch.equal(md.cpu()[0, pages[d // 64], 0, d % 64], m[0, pages[s // 64], 0, s % 64])


def test_evict_reports_a_missing_page_and_refuses():
    from mynah_slm_b200.ops import evict
    from mynah_slm_b200.ops.kernels import PageTableView
    from mynah_slm_b200.ops.lib import KernelError
    step, k, v, m, _ = _evict_case(7, [300, 100], 2, 2, 64, 64, BF16)
    k, v, m = k.to(DEV), v.to(DEV), m.to(DEV)
    ids = step.pages.ids.clone()
    ids[1] = 99999
    evict.cache_evict(k, v, m, step, PageTableView(step.pages.indptr, ids, step.pages.base, step.pages.n_pages), 80, 10)
    torch.cuda.synchronize()
    assert step.status.item() & 1

    def bad(**kw):
        a = dict(k_caches=k, v_caches=v, masses=m, ctx=step, pages=step.pages, keep=64, recent=8, first=2)
        a.update(kw)
        with pytest.raises(KernelError):
            evict.cache_evict(**a)
    bad(keep=0)
    bad(recent=-1)
    bad(first=60)
    bad(masses=m[:1])
    bad(masses=m.double())
    bad(k_caches=k[0])
    bad(v_caches=v[:, :, :1])
    bad(v_caches=v.float())
    bad(out_pages=PageTableView(step.pages.indptr, step.pages.ids, step.pages.base, 3))
    bad(out_pages=PageTableView(step.pages.indptr.long(), step.pages.ids, step.pages.base, step.pages.n_pages))
