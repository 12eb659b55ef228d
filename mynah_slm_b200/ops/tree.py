"""Trees of drafted tokens over the paged cache: the attention of a step that brings a tree for every sequence, and the
acceptance of a tree's path with the move of its rows.

A step that checks drafted tokens brings, for each sequence, a tree: row 0 is the token that was sampled last, every other row
hangs on an earlier row (`parents`, -1 for none). All rows' keys and values are written to the cache behind what it holds, row
past + i for the tree's row i, but rotated for their positions, past + depth. Every row attends to what was held and to its
ancestors. What the model then chooses behind every row decides which path goes on (`tree_commit`): the path's rows move to
past + 0, 1, 2, ..., where a sequence that had taken the tokens one by one would have them.
"""
from __future__ import annotations

from functools import lru_cache
from struct import Struct
from typing import Optional, Sequence

import numpy as np
import torch

from ..cache.pages import PAGE_TOKENS
from . import lib
from .kernels import MAX_HEAD_DIM, PageTableView
from .lib import KernelError, call, code, stream_on

_LEAST, _MOST = 2.0 ** -120, 2.0 ** 120      # a score scale, which the kernels hold in fp32, times log2(e)
_I32 = torch.int32
# the arguments of the C entries, which take them as one struct
_TREE_CALL = Struct("@2P9i7P2iPifPq2P")
_COMMIT_CALL = Struct("@3P3i5Pi2P4i5P")


def tree_rows(parents: Sequence[int], words: Optional[int] = None) -> tuple[np.ndarray, np.ndarray]:
    """What a step needs to know of a tree given as every row's parent (an earlier row, or -1): (depths int32 [n], mask words
    int64 [n, words]); bit j of row i's words (bit j % 64 of word j // 64) says that row j is row i or an ancestor of it."""
    n = len(parents)
    need = max(1, -(-n // 64))
    words = need if words is None else int(words)
    if words < need:
        raise KernelError(f"tree_rows: {words} mask words for a tree of {n} rows, {need} are needed")
    depth = np.zeros((n,), dtype=np.int32)
    bits = np.zeros((n, words), dtype=np.uint64)
    for i, p in enumerate(parents):
        p = int(p)
        if not -1 <= p < i:
            raise KernelError(f"tree_rows: row {i} hangs on row {p}, which is not before it")
        if p >= 0:
            depth[i] = depth[p] + 1
            bits[i] = bits[p]
        bits[i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return depth, bits.view(np.int64)


def check_rows(who: str, q: torch.Tensor, out: torch.Tensor, ctx, H: int, KV: int, HD: int, k_cache: torch.Tensor,
               v_cache: torch.Tensor, pages: PageTableView, scale: float) -> tuple[int, int, int, int, int]:
    """What the attention of a few rows a sequence asks of its arguments. Returns q's type code and device, its rows, and the row
    strides of q and the output. (Every call pays for this in full: few and cheap lookups.)"""
    index, dt = q.get_device(), q.dtype
    if index < 0 or index != torch.cuda.current_device():
        raise KernelError(f"{who}: q is not on the current CUDA device")
    if KV < 1 or H < 1 or H % KV:
        raise KernelError(f"{who}: {H} heads over {KV} kv heads")
    if HD < 1 or HD % 8 or HD > MAX_HEAD_DIM:
        raise KernelError(f"{who}: head_dim {HD} is no multiple of 8 up to {MAX_HEAD_DIM}")
    if scale != 0.0 and not _LEAST <= scale <= _MOST:
        raise KernelError(f"{who}: the score scale {scale} is not between 2^-120 and 2^120, nor 0 for 1 / sqrt(head_dim)")
    dcode = code(dt)
    T, ldq = _rows_of(who, q, H * HD)
    n_out, ldo = _rows_of(who, out, H * HD)
    if out.dtype is not dt or out.get_device() != index or n_out < T:
        raise KernelError(f"{who}: the output is {tuple(out.shape)} {out.dtype} on {out.device}, q {tuple(q.shape)} {dt} on {q.device}")
    if T and _over(q.data_ptr(), out.data_ptr(), T, ldq, ldo, H * HD, q.element_size()):
        raise KernelError(f"{who}: the output lies over q, which is read until the end")
    cache = (KV, PAGE_TOKENS, HD)
    for t in (k_cache, v_cache):
        shape = t.shape
        if t.dtype is not dt or t.get_device() != index or len(shape) != 4 or shape[1:] != cache \
                or shape[0] < pages.n_pages or not t.is_contiguous():
            raise KernelError(f"{who}: the cache must be contiguous [{pages.n_pages}, {KV}, {PAGE_TOKENS}, {HD}] of q's type and device, "
                              f"got {tuple(t.shape)} {t.dtype} on {t.device}")
    if ctx.B < 0 or ctx.max_q_len < 0:
        raise KernelError(f"{who}: {ctx.B} sequences of up to {ctx.max_q_len} rows")
    check_lists(who, index, ctx.B, ctx.cu_q, ctx.kv_len, pages, ctx.status)
    return dcode, index, T, ldq, ldo


def _rows_of(who: str, t: torch.Tensor, width: int) -> tuple[int, int]:
    """(rows, row stride) of q or the output."""
    if t.dim() == 2:
        n, w = t.shape
        ld, one = t.stride()
        if w >= width and one == 1 and (n < 2 or width <= ld < 1 << 31):
            return n, ld if n > 1 else w
    raise KernelError(f"{who}: q and the output must be rows of at least {width} values, one row behind the other, got "
                      f"{tuple(t.shape)} with strides {t.stride()}")


def _over(q: int, out: int, T: int, ldq: int, ldo: int, width: int, es: int) -> bool:
    """Whether T rows of `width` values at two addresses may share memory. Columns of one buffer may lie side by side."""
    if q + ((T - 1) * ldq + width) * es <= out or out + ((T - 1) * ldo + width) * es <= q:
        return False
    if ldq != ldo:
        return True
    apart = (out - q) % (ldq * es)
    return apart < width * es or apart > (ldq - width) * es


def check_lists(who: str, index: int, B: int, cu_q: Optional[torch.Tensor], kv_len: torch.Tensor, pages: PageTableView, status: torch.Tensor) -> None:
    for t, n in ((cu_q, B + 1), (kv_len, B), (pages.indptr, B + 1), (pages.base, B), (pages.ids, 0), (status, 1)):
        if t is not None and (t.dtype is not _I32 or t.get_device() != index or t.numel() < n or not t.is_contiguous()):
            raise KernelError(f"{who}: cu_q, kv_len, the page lists and the status word must be contiguous int32 on cuda:{index} for {B} "
                              f"sequences, got {tuple(t.shape)} {t.dtype} on {t.device}")


def row_scratch(who: str, scratch: Optional[torch.Tensor], need: int, status: torch.Tensor) -> torch.Tensor:
    dev = status.device
    if scratch is None:
        return status.new_empty(need)                          # (32-bit words; torch.empty takes a us more)
    if scratch.dtype != torch.float32 or scratch.device != dev or not scratch.is_contiguous() or scratch.numel() < need:
        raise KernelError(f"{who}: scratch must be at least {need} contiguous float32 on {dev}")
    return scratch


@lru_cache(maxsize=256)
def _tree_scratch(T: int, B: int, max_q_len: int, H: int, KV: int, HD: int, dcode: int, n_ids: int, aligned: int) -> int:
    return int(lib.load().mynah_attn_tree_scratch_floats(T, B, max_q_len, H, KV, HD, dcode, n_ids, aligned))


def rows_aligned(q: torch.Tensor, out: torch.Tensor, ldq: int, ldo: int) -> int:
    """Whether the rows of q and of the output begin at whole 16 bytes: the tensor cores take such a call."""
    es = q.element_size()
    return 0 if (q.data_ptr() | out.data_ptr() | ldq * es | ldo * es) & 15 else 1


def attn_tree_scratch_floats(T: int, B: int, max_q_len: int, H: int, KV: int, HD: int, dtype: torch.dtype) -> int:
    """Words that serve a call of this shape whatever its page lists and alignment are (most calls need fewer)."""
    return _tree_scratch(T, B, max_q_len, H, KV, HD, code(dtype), -1, -1)


def attn_tree(q: torch.Tensor, out: torch.Tensor, ctx, H: int, KV: int, HD: int, k_cache: torch.Tensor, v_cache: torch.Tensor,
              pages: PageTableView, masks: torch.Tensor, scale: float = 0.0, scratch: Optional[torch.Tensor] = None) -> None:
    """Attention of a step's rows over the paged cache, which holds the rows' own keys and values already: with past = kv_len -
    n_q, row i of a sequence sees every cached row below past, and row past + j where bit j of its mask words is set (`tree_rows`
    makes the words of a tree; any other mask will do, a row that sees nothing gives zeros). Query head h reads kv head
    h // (H / KV). `q` and `out` are rows with head h in columns [h HD, (h + 1) HD), and may be wider (columns of one
    buffer side by side too, but never over one another); rows of `out` behind the
    last sequence are left as they are. masks: int64 [T, words]; rows of a tree beyond 64 * words are seen by nobody. scale 0:
    1 / sqrt(HD), else 2^-120 to 2^120. ctx: the step's description (B, max_q_len, cu_q, kv_len, status; max_q_len only
    sizes the tiles, a longer sequence is served too). Rows of the cache that a row does not see
    have no influence on it, whatever they hold. float32 and bfloat16, heads of any multiple of 8 up to 256; bfloat16 heads of 64
    and 128 run on the tensor cores. `scratch`: attn_tree_scratch_floats fp32 words, taken from torch's allocator unless given."""
    dt, index, T, ldq, ldo = check_rows("attn_tree", q, out, ctx, H, KV, HD, k_cache, v_cache, pages, scale)
    if masks.dtype is not torch.int64 or masks.dim() != 2 or masks.shape[0] < T or masks.shape[1] < 1 or not masks.is_contiguous() \
            or masks.get_device() != index:
        raise KernelError(f"attn_tree: the masks must be contiguous int64 [{T}, words] on {q.device}, got {tuple(masks.shape)} {masks.dtype}")
    if T == 0 or ctx.B == 0:
        return
    n_ids = pages.ids.numel()
    scratch = row_scratch("attn_tree", scratch, _tree_scratch(T, ctx.B, ctx.max_q_len, H, KV, HD, dt, n_ids, rows_aligned(q, out, ldq, ldo)), ctx.status)
    call("mynah_attn_tree", _TREE_CALL.pack(
        q.data_ptr(), out.data_ptr(), dt, T, ctx.B, ctx.max_q_len, H, KV, HD, ldq, ldo, k_cache.data_ptr(), v_cache.data_ptr(), ctx.cu_q.data_ptr(),
        ctx.kv_len.data_ptr(), pages.indptr.data_ptr(), pages.ids.data_ptr(), pages.base.data_ptr(), pages.n_pages, n_ids, masks.data_ptr(), masks.shape[1],
        scale, scratch.data_ptr(), scratch.numel(), ctx.status.data_ptr(), stream_on(index)))


def check_layers(who: str, k_caches: torch.Tensor, v_caches: torch.Tensor, pages: PageTableView) -> int:
    """What the operators over all layers' rows ask of a storage group. Returns its device."""
    ks, vs, index = k_caches.shape, v_caches.shape, k_caches.get_device()
    if index < 0 or index != torch.cuda.current_device():
        raise KernelError(f"{who}: the cache is not on the current CUDA device")
    if len(ks) != 5 or len(vs) != 5 or ks[1] != pages.n_pages or ks[3] != PAGE_TOKENS or ks[:4] != vs[:4] or k_caches.dtype is not v_caches.dtype \
            or v_caches.get_device() != index or not k_caches.is_contiguous() or not v_caches.is_contiguous():
        raise KernelError(f"{who}: the cache must be contiguous [layers, {pages.n_pages}, kv heads, {PAGE_TOKENS}, head], got K {tuple(ks)} "
                          f"{k_caches.dtype}, V {tuple(vs)} {v_caches.dtype}")
    return index


def tree_commit(tokens: torch.Tensor, parents: torch.Tensor, chosen: torch.Tensor, ctx, k_caches: torch.Tensor, v_caches: torch.Tensor,
                pages: PageTableView) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The path of every sequence's tree that the model's choices accept, and the move of its rows in all layers, in one launch.

    tokens, parents, chosen: int32 [T], the step's tokens, every row's parent within its sequence (-1: none; a parent that is
    not an earlier row counts as none), and the token chosen behind every row (the most likely one, or one drawn). From a
    sequence's row 0 on, a row goes on to its lowest child whose token was chosen behind it. Cached row past + path[i] becomes
    row past + i in every layer of k_caches, v_caches [layers, n_pages, kv heads, 64, head] (a storage group of the cache), past =
    kv_len - n_q. Returns int32 (path [T]: the path's rows from every sequence's first place on, -1 behind them; count [B]; next
    [B]: what was chosen behind the path's last row). A sequence without rows has count 0 and next -1. Trees of up to 4,096 rows;
    ctx.max_q_len is the longest one's (a longer one is refused through the status word, with count 0)."""
    index = check_layers("tree_commit", k_caches, v_caches, pages)
    T = tokens.numel()
    for t in (tokens, parents, chosen):
        if t.dtype is not _I32 or t.get_device() != index or t.dim() != 1 or t.numel() < T or not t.is_contiguous():
            raise KernelError(f"tree_commit: tokens, parents and chosen tokens must be {T} contiguous int32 on cuda:{index}")
    if not 0 <= ctx.max_q_len <= 4096:
        raise KernelError(f"tree_commit: trees of {ctx.max_q_len} rows, 4096 are the most")
    check_lists("tree_commit", index, ctx.B, ctx.cu_q, ctx.kv_len, pages, ctx.status)
    path, count, after = tokens.new_empty(T), tokens.new_empty(ctx.B), tokens.new_empty(ctx.B)       # (torch.empty takes a us more)
    E, _, KV, _, HD = k_caches.shape
    es = k_caches.element_size()
    call("mynah_tree_commit", _COMMIT_CALL.pack(
        tokens.data_ptr(), parents.data_ptr(), chosen.data_ptr(), T, ctx.B, ctx.max_q_len, ctx.cu_q.data_ptr(), ctx.kv_len.data_ptr(),
        pages.indptr.data_ptr(), pages.ids.data_ptr(), pages.base.data_ptr(), pages.n_pages, k_caches.data_ptr(), v_caches.data_ptr(), E, KV, HD * es,
        v_caches.shape[4] * es, path.data_ptr(), count.data_ptr(), after.data_ptr(), ctx.status.data_ptr(), stream_on(index)))
    return path, count, after
