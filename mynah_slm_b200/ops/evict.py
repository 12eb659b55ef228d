"""A bounded cache: attention that adds up the weight every cached row gets, and the eviction of the rows that got least.

Every cached row has, in every layer and kv head, a sum: the softmax weight that all tokens so far have given it, over the query
heads of the kv head. When a sequence holds more rows than it may keep, each layer and kv head keeps its first few rows, its
most recent ones, and of those between them the ones with the greatest sums; the rows that stay move together, in order, and the
sequence goes on behind them. (The rows' positions are in the keys already: a cache whose rows have moved is attended to as it
is, while the tokens that follow are rotated for their true positions.)
"""
from __future__ import annotations

from functools import lru_cache
from struct import Struct
from typing import Optional

import torch

from ..cache.pages import PAGE_TOKENS
from . import lib
from .kernels import PageTableView
from .lib import KernelError, call, code, stream_on
from .tree import check_layers, check_lists, check_rows, row_scratch, rows_aligned

# the arguments of the C entries, which take them as one struct
_MASS_CALL = Struct("@3P9i7P2ifPq2P")
_EVICT_CALL = Struct("@3P6i4Pi3P4i4P")


@lru_cache(maxsize=256)
def _mass_scratch(T: int, B: int, max_q_len: int, H: int, KV: int, HD: int, dcode: int, n_ids: int, aligned: int) -> int:
    return int(lib.load().mynah_attn_mass_scratch_floats(T, B, max_q_len, H, KV, HD, dcode, n_ids, aligned))


def attn_mass_scratch_floats(T: int, B: int, max_q_len: int, H: int, KV: int, HD: int, dtype: torch.dtype, n_ids: int) -> int:
    """Words that serve a call of this shape; n_ids: entries of the page lists (a call whose rows are 16-byte aligned may need fewer)."""
    return _mass_scratch(T, B, max_q_len, H, KV, HD, code(dtype), n_ids, -1)


def attn_mass(q: torch.Tensor, out: torch.Tensor, mass: torch.Tensor, ctx, H: int, KV: int, HD: int, k_cache: torch.Tensor,
              v_cache: torch.Tensor, pages: PageTableView, scale: float = 0.0, scratch: Optional[torch.Tensor] = None) -> None:
    """Causal attention of a step's rows (a token a sequence, pieces of prompts, whole prompts) over the paged cache, which holds
    the rows' own keys and values already, as `attn_tree` with every row seeing the rows up to itself; and the sums of the weights:
    mass [n_pages, KV, 64] fp32 gets, at every cached row of the step's sequences, the weight that the step's rows and the kv
    head's query heads give it, added to what it holds for rows that were there before the step, in place of it for the step's own
    (so nothing has to be cleared when a page is taken). Other rows' sums are left as they are. No sequence may have more than
    ctx.max_q_len rows in the step: one that has (a replay with other lengths) is refused through the status word, its outputs and
    sums left alone. The order of the sums does not
    depend on timing, provided that no page is in two sequences' lists (a shared page's sums would be written by both)."""
    dt, index, T, ldq, ldo = check_rows("attn_mass", q, out, ctx, H, KV, HD, k_cache, v_cache, pages, scale)
    if mass.dtype is not torch.float32 or mass.get_device() != index or not mass.is_contiguous() or mass.dim() != 3 \
            or mass.shape[1:] != (KV, PAGE_TOKENS) or mass.shape[0] < pages.n_pages:
        raise KernelError(f"attn_mass: the sums must be contiguous float32 [{pages.n_pages}, {KV}, {PAGE_TOKENS}] on {q.device}, "
                          f"got {tuple(mass.shape)} {mass.dtype}")
    if T == 0 or ctx.B == 0:
        return
    n_ids = pages.ids.numel()
    need = _mass_scratch(T, ctx.B, ctx.max_q_len, H, KV, HD, dt, n_ids, rows_aligned(q, out, ldq, ldo))
    scratch = row_scratch("attn_mass", scratch, need, ctx.status)
    call("mynah_attn_mass", _MASS_CALL.pack(
        q.data_ptr(), out.data_ptr(), mass.data_ptr(), dt, T, ctx.B, ctx.max_q_len, H, KV, HD, ldq, ldo, k_cache.data_ptr(), v_cache.data_ptr(),
        ctx.cu_q.data_ptr(), ctx.kv_len.data_ptr(), pages.indptr.data_ptr(), pages.ids.data_ptr(), pages.base.data_ptr(), pages.n_pages, n_ids, scale,
        scratch.data_ptr(), scratch.numel(), ctx.status.data_ptr(), stream_on(index)))


def cache_evict(k_caches: torch.Tensor, v_caches: torch.Tensor, masses: torch.Tensor, ctx, pages: PageTableView, keep: int, recent: int,
                first: int = 0, out_pages: Optional[PageTableView] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Cuts every sequence that holds more than `keep` rows down to `keep`, in every layer and kv head on its own: the first
    `first` rows and the last `recent` stay, and of those between them the keep - first - recent with the greatest sums (the lower
    row where sums are equal; a NaN counts as the greatest). The rows that stay become rows 0, 1, 2, ..., in order, with their
    sums: in the same pages, or in those of `out_pages`, whose lists must have no page in common with `pages`' (sequences of no
    more than `keep` rows are then copied whole). No page may be in two sequences' lists, unless its rows go to `out_pages`.

    k_caches, v_caches [layers, n_pages, kv heads, 64, head], masses [layers, n_pages, kv heads, 64] fp32, ctx.kv_len: the rows
    held. Returns int32 (kept [layers, B, kv heads, keep]: the rows that stayed, ascending, -1 behind them; kv_len [B])."""
    index = check_layers("cache_evict", k_caches, v_caches, pages)
    E, n_pages, KV, _, HD = k_caches.shape
    if masses.dtype is not torch.float32 or masses.get_device() != index or not masses.is_contiguous() or masses.shape != (E, n_pages, KV, PAGE_TOKENS):
        raise KernelError(f"cache_evict: the sums must be contiguous float32 {(E, n_pages, KV, PAGE_TOKENS)} on cuda:{index}, "
                          f"got {tuple(masses.shape)} {masses.dtype}")
    keep, recent, first = int(keep), int(recent), int(first)
    if not 1 <= keep < 1 << 31 or recent < 0 or first < 0 or recent + first > keep:
        raise KernelError(f"cache_evict: {first} first and {recent} recent rows do not fit the {keep} that are kept")
    check_lists("cache_evict", index, ctx.B, None, ctx.kv_len, pages, ctx.status)
    same = out_pages is None
    if same:
        out_pages = pages
    else:
        check_lists("cache_evict", index, ctx.B, None, ctx.kv_len, out_pages, ctx.status)
        if out_pages.n_pages != n_pages:
            raise KernelError(f"cache_evict: the out pages are of a pool of {out_pages.n_pages}, the pages of one of {n_pages}")
    es = k_caches.element_size()
    kept, new_len = ctx.kv_len.new_empty((E, ctx.B, KV, keep)), ctx.kv_len.new_empty(ctx.B)
    if E == 0 or ctx.B == 0:
        return kept, new_len
    call("mynah_cache_evict", _EVICT_CALL.pack(
        k_caches.data_ptr(), v_caches.data_ptr(), masses.data_ptr(), E, ctx.B, KV, n_pages, HD * es, v_caches.shape[4] * es, ctx.kv_len.data_ptr(),
        pages.indptr.data_ptr(), pages.ids.data_ptr(), pages.base.data_ptr(), pages.ids.numel(), out_pages.indptr.data_ptr(), out_pages.ids.data_ptr(),
        out_pages.base.data_ptr(), same, keep, recent, first, kept.data_ptr(), new_len.data_ptr(), ctx.status.data_ptr(), stream_on(index)))
    return kept, new_len
