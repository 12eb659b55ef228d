"""Trees of drafted tokens on the host: depths, mask words, refusals that need no device."""
import random

import numpy as np
import pytest
import torch

from mynah_slm_b200.ops.lib import KernelError
from mynah_slm_b200.ops.tree import tree_rows


def test_depths_and_ancestors():
    depth, words = tree_rows([-1, 0, 0, 1, 3, 2, -1])
    assert depth.tolist() == [0, 1, 1, 2, 3, 2, 0]
    assert [bin(w) for w in words[:, 0]] == ["0b1", "0b11", "0b101", "0b1011", "0b11011", "0b100101", "0b1000000"]


def test_long_trees_take_more_words():
    n = 200
    depth, words = tree_rows([-1] + list(range(n - 1)))
    assert words.shape == (n, 4) and words.dtype == np.int64 and depth[-1] == n - 1
    for i in (0, 62, 63, 64, 127, 128, 199):
        bits = [(int(words[i, j // 64]) >> (j % 64)) & 1 for j in range(256)]
        assert bits == [1 if j <= i else 0 for j in range(256)]
    assert tree_rows([-1], 3)[1].tolist() == [[1, 0, 0]]
    depth, words = tree_rows([])
    assert depth.shape == (0,) and words.shape == (0, 1)


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 2, 0], [-2]])
def test_parents_that_are_not_before_their_rows_are_refused(parents):
    with pytest.raises(KernelError):
        tree_rows(parents)


def test_too_few_words_are_refused():
    with pytest.raises(KernelError):
        tree_rows([-1] + [0] * 64, 1)


def test_tensors_that_are_not_on_a_device_are_refused():
    from types import SimpleNamespace
    from mynah_slm_b200.ops import evict, tree
    t = torch.zeros
    i32 = lambda n: t(n, dtype=torch.int32)  # noqa: E731
    pages = SimpleNamespace(indptr=i32(2), ids=i32(1), base=i32(1), n_pages=1)
    ctx = SimpleNamespace(B=1, max_q_len=1, cu_q=i32(2), kv_len=i32(1), status=i32(1))
    k = t((1, 1, 64, 8))
    with pytest.raises(KernelError):
        tree.attn_tree(t((1, 8)), t((1, 8)), ctx, 1, 1, 8, k, k, pages, t((1, 1), dtype=torch.int64))
    with pytest.raises(KernelError):
        evict.attn_mass(t((1, 8)), t((1, 8)), t((1, 1, 64)), ctx, 1, 1, 8, k, k, pages)
    with pytest.raises(KernelError):
        evict.cache_evict(k[None], k[None], t((1, 1, 1, 64)), ctx, pages, 2, 1)
    with pytest.raises(KernelError):
        tree.tree_commit(i32(1), i32(1), i32(1), ctx, k[None], k[None], pages)


def test_outputs_over_the_queries_are_told_from_those_beside_them():
    """Against every byte that the rows take."""
    from mynah_slm_b200.ops.tree import _over
    rng = random.Random(3)
    for _ in range(3000):
        es, width, T = rng.choice([2, 4]), rng.randrange(1, 9), rng.randrange(1, 5)
        ldq = width + rng.randrange(0, 20)
        ldo = ldq if rng.random() < 0.7 else width + rng.randrange(0, 20)
        q, out = 1000 * es, (1000 + rng.randrange(-40, 41)) * es
        taken = [{at + (r * ld + c) * es for r in range(T) for c in range(width)} for at, ld in ((q, ldq), (out, ldo))]
        shared = bool(taken[0] & taken[1])
        if ldq == ldo:
            # (equal pitches: exact but for rows that only others of the buffer, not these T, would meet)
            assert _over(q, out, T, ldq, ldo, width, es) or not shared
            endless = [{at + (r * ld + c) * es for r in range(-60, 60) for c in range(width)} for at, ld in ((q, ldq), (out, ldo))]
            if not endless[0] & endless[1]:
                assert not _over(q, out, T, ldq, ldo, width, es)
        elif shared:
            assert _over(q, out, T, ldq, ldo, width, es)
