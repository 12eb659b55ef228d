"""Drafted trees from a sequence's own text, the generation loop that takes several tokens a step, and books that are cut, on the host."""
import random

import pytest

from mynah_slm_b200.cache.pages import CacheError, GroupPlan, SequencePages
from mynah_slm_b200.engine.draft import Lookup
from mynah_slm_b200.engine.generate import tokens_held, Request, generate, plan_batches


def test_a_tree_is_one_and_stays_within_its_room():
    rng = random.Random(1)
    for _ in range(200):
        text = [rng.randrange(4) for _ in range(rng.randrange(1, 60))]
        room = rng.randrange(0, 20)
        tokens, parents = Lookup(text).tree(room)
        assert tokens[0] == text[-1] and parents[0] == -1 and 1 <= len(tokens) == len(parents) <= 1 + room
        assert all(0 <= p < i for i, p in enumerate(parents) if i)
        kids = [(p, t) for p, t in zip(parents, tokens)]
        assert len(set(kids)) == len(kids)                 # no child twice
        for i in range(1, len(tokens)):                    # every path continues the text as it went on somewhere before
            path = []
            at = i
            while at > 0:
                path.append(tokens[at])
                at = parents[at]
            run = [text[-1]] + path[::-1]
            assert any(text[j:j + len(run)] == run for j in range(len(text)))


def test_text_that_repeats_itself_is_drafted():
    text = [1, 2, 3, 4, 5, 6, 7, 1, 2, 3]
    assert Lookup(text).tree(4) == ([3, 4, 5, 6, 7], [-1, 0, 1, 2, 3])
    two = [1, 2, 9, 1, 2, 8, 1, 2]
    tokens, parents = Lookup(two).tree(6)
    assert (tokens[1], parents[1]) == (8, 0) and 9 in [t for t, p in zip(tokens, parents) if p == 0]
    assert Lookup([5]).tree(8) == ([5], [-1])
    grown = Lookup([1, 2, 3])
    grown.extend([4, 1, 2])
    assert grown.tree(2) == Lookup([1, 2, 3, 4, 1, 2]).tree(2)


class Drafting:
    """A model that counts up modulo 7; every step gains as many tokens as its room and its drafts allow."""
    max_positions, drafts = 64, 3

    def __init__(self):
        self.steps = 0

    def free_tokens(self): return 4096
    def open(self, i, prompt): return i
    def close(self, slot): pass
    def prefill(self, slots, prompts): return [(p[-1] + 1) % 7 for p in prompts]
    def decode(self, slots, tokens): raise AssertionError("the drafted step is taken")

    def decode_drafted(self, slots, last, rooms):
        self.steps += 1
        assert all(r >= 1 for r in rooms)
        return [[(t + 1 + k) % 7 for k in range(min(1 + self.drafts, r))] for t, r in zip(last, rooms)]


def test_the_loop_takes_several_tokens_a_step():
    backend = Drafting()
    out = generate(backend, [Request([0], 9), Request([3, 4], 2), Request([1] * 60, 30)])
    assert out[0].tokens == [1, 2, 3, 4, 5, 6, 0, 1, 2] and out[0].finish_reason == "length"
    assert out[1].tokens == [5, 6] and out[1].finish_reason == "length"
    assert len(out[2].tokens) == 5 and out[2].finish_reason == "context"      # 60 positions, 4 more, one behind the last
    assert backend.steps == 2
    out = generate(Drafting(), [Request([0], 20)], stop_ids=[3])
    assert out[0].tokens == [1, 2] and out[0].finish_reason == "stop" and out[0].produced == 3


def test_batches_go_by_what_a_backend_holds():
    reqs = [Request([1] * 100, 1000), Request([1] * 100, 1000)]
    assert plan_batches(reqs, 8, 256, 4096, rows_held=lambda p, n: 128) == [[0, 1]]


def test_books_that_are_cut_give_their_pages_back():
    books = SequencePages([GroupPlan(1, 8, None), GroupPlan(1, 8, None)], 8, 2)
    a, b = books.open(), books.open()
    books.reserve(a, 300)
    books.commit(a, 290)
    before = books.held(a, 1)[0]
    books.shorten(a, 130)
    assert books.length[a] == 130 and books.held(a, 1) == (before[:3], 0)
    assert books.pools[0].n_free == 5
    books.reserve(b, 300)                                   # what was given back is there for others
    with pytest.raises(CacheError):
        books.shorten(a, 131)
    with pytest.raises(CacheError):
        books.shorten(a, -1)
    books.shorten(a, 130)
    books.shorten(a, 0)
    assert books.length[a] == 0 and books.held(a, 0) == ([], 0)
    with pytest.raises(CacheError):
        books.shorten(7, 0)
    windowed = SequencePages([GroupPlan(1, 8, 64)], 8, 2)
    s = windowed.open()
    windowed.reserve(s, 10)
    windowed.commit(s, 10)
    with pytest.raises(CacheError):
        windowed.shorten(s, 5)


def test_drafts_need_no_cache_of_their_own():
    """A request that fits without drafts fits with them: no step's tree reaches beyond the rows that the request may hold."""
    from types import SimpleNamespace
    from mynah_slm_b200.engine.api import EngineBackend
    from mynah_slm_b200.engine.engine import TreeResult
    from mynah_slm_b200.sampling.sampler import SamplingParams
    held, most = {}, {}

    def step_tree(entries):
        out = []
        for e in entries:
            most[e.slot] = max(most.get(e.slot, 0), held[e.slot] + len(e.tokens))
            path = [0]                                     # the first child of every row, all the way down
            while path[-1] in e.parents:
                path.append(list(e.parents).index(path[-1]))
            held[e.slot] += len(path)
            out.append(TreeResult([e.tokens[i] for i in path[1:]], 5))
        return out
    engine = SimpleNamespace(spec=SimpleNamespace(max_positions=4096), keep=None, use_graphs=False, graph_safe=False, step_tree=step_tree,
                             sampler=SimpleNamespace(set_params=lambda p: None))
    for drafts in (1, 8, 200):
        b = EngineBackend(engine, SamplingParams.greedy(), drafts)
        for prompt, new in ((40, 24), (1, 63), (100, 28), (5, 1)):
            assert b.rows_held(prompt, new) == tokens_held(prompt, new, 4096)
            text = [1, 5, 2, 5, 3] * 20
            b._lookups[0] = Lookup(text[:prompt])
            held[0], most[0], produced, last = prompt, 0, 1, 5
            while produced < new:
                got = b.decode_drafted([0], [last], [new - produced])[0]
                assert 1 <= len(got) <= new - produced
                produced, last = produced + len(got), got[-1]
            assert most[0] <= prompt + new - 1
