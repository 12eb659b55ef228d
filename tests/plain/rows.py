"""Attention of a few rows a sequence over the paged cache, the sums of its weights, the choice of rows that stay and the
acceptance of a tree, in 64 bits and from their definitions, with the bounds that the kernels' roundings allow."""
from __future__ import annotations

from dataclasses import dataclass

import torch

PAGE = 64
F32 = 2.0 ** -24          # a rounding to fp32, relative


@dataclass
class Step:
    """A ragged step over a paged cache (all tensors on the device, the oracle takes them to the host)."""
    B: int
    max_q_len: int
    cu_q: torch.Tensor
    kv_len: torch.Tensor
    status: torch.Tensor
    q_lens: list
    past: list
    pages: object
    lists: list            # page ids of every sequence


def make_step(rows, past, device, gen, spare=3, lists=None):
    from mynah_slm_b200.ops.kernels import PageTableView
    held = [p + n for p, n in zip(past, rows)]
    counts = [-(-h // PAGE) for h in held]
    n_pages = sum(counts) + spare
    if lists is None:
        perm = torch.randperm(n_pages, generator=gen).tolist()
        lists = [[perm.pop() for _ in range(c)] for c in counts]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    cu, indptr = [0], [0]
    for n, c in zip(rows, counts):
        cu.append(cu[-1] + n)
        indptr.append(indptr[-1] + c)
    pages = PageTableView(i32(indptr), i32([p for l in lists for p in l] or [0]), i32([0] * len(rows)), n_pages)
    return Step(len(rows), max(rows + [0]), i32(cu), i32(held), torch.zeros(1, dtype=torch.int32, device=device), list(rows), list(past),
                pages, lists)


def cached_rows(cache, pages, n, g):
    """Rows 0 .. n - 1 of a kv head, [n, width]."""
    return cache[torch.tensor(pages, dtype=torch.long), g].reshape(-1, *cache.shape[3:])[:n] if n else cache[:0, g].reshape(0, *cache.shape[3:])


def attention(step, q, k, v, H, scale, sees, p_bits, acc):
    """sees[b]: bool [n_q, kv_len] of sequence b. q [T, H HD], k and v [pages, KV, 64, HD] on the host, in the run's type.
    Returns (out [T, H, HD], bound of its error before the last rounding, weights' sums per sequence [KV, kv_len] and their
    bounds). p_bits: relative rounding of a weight before it meets the values (0 where it stays fp32); acc: relative error of one
    addition in the accumulations (fp32's, or twice that where a tensor core cuts instead of rounding).

    The bounds: a score of HD products is off by at most (HD + 2) acc A, A = scale sum |q k|, the subtraction of the reference
    and the base change by 4 acc (A + 8), which its exponential turns into a relative error of the weight (times ln 2 at most
    1); the exponential itself by 2^-21; the sum of N weights by N acc; the quotient and a join of chunks by 16 acc. The
    output's sum of N products adds N acc and the weights' own roundings, all relative to sum w |v|."""
    KV, HD = k.shape[1], k.shape[3]
    G = H // KV
    T = q.shape[0]
    out = torch.zeros((T, H, HD), dtype=torch.float64)
    bound = torch.zeros((T, H, HD), dtype=torch.float64)
    sums, sum_bounds = [], []
    at = 0
    for b, (n, p) in enumerate(zip(step.q_lens, step.past)):
        held = p + n
        total = torch.zeros((KV, held), dtype=torch.float64)
        slack = torch.zeros((KV, held), dtype=torch.float64)
        for g in range(KV):
            kk = cached_rows(k, step.lists[b], held, g).double()
            vv = cached_rows(v, step.lists[b], held, g).double()
            for h in range(g * G, (g + 1) * G):
                qq = q[at:at + n, h * HD:(h + 1) * HD].double()
                for i in range(n):
                    r = sees[b][i].nonzero()[:, 0]
                    if r.numel() == 0:
                        continue
                    z = kk[r] @ qq[i] * scale
                    w = torch.softmax(z, 0)
                    A = (kk[r].abs() @ qq[i].abs() * scale).max()
                    N = r.numel()
                    rel = (HD + 2) * acc * A * 2 + 8 * acc * (A + 8) + 2.0 ** -20 + (N + 16) * acc
                    out[at + i, h] = w @ vv[r]
                    bound[at + i, h] = (w @ vv[r].abs()) * (rel + p_bits + N * acc)
                    total[g, r] += w
                    slack[g, r] += w * (rel + (n * G + 4) * acc)
        sums.append(total)
        sum_bounds.append(slack)
        at += n
    return out, bound, sums, sum_bounds


def causal(step):
    return [torch.ones((n, p + n), dtype=torch.bool).tril(p) for n, p in zip(step.q_lens, step.past)]


def by_words(step, masks):
    """masks int64 [T, words] on the host."""
    seen, at = [], 0
    for n, p in zip(step.q_lens, step.past):
        s = torch.ones((n, p + n), dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                word = masks[at + i, j // 64].item() if j // 64 < masks.shape[1] else 0
                s[i, p + j] = bool((word >> (j % 64)) & 1)
        seen.append(s)
        at += n
    return seen


def kept_rows(sums, n, keep, recent, first):
    """sums: list of n numbers. The rows that stay, ascending."""
    if n <= keep:
        return list(range(n))
    key = lambda r: (0 if sums[r] != sums[r] else 1, -sums[r] if sums[r] == sums[r] else 0.0, r)  # noqa: E731
    middle = sorted(range(first, n - recent), key=key)[: keep - first - recent]
    return list(range(first)) + sorted(middle) + list(range(n - recent, n))


def accepted(tokens, parents, chosen):
    """Lists of one sequence's tree -> (path, next)."""
    if not tokens:
        return [], -1
    path = [0]
    while True:
        at = path[-1]
        nxt = [c for c in range(1, len(tokens)) if parents[c] == at and c > at and tokens[c] == chosen[at]]
        if not nxt:
            return path, chosen[at]
        path.append(nxt[0])
